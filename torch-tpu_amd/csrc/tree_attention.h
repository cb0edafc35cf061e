// Attention of new tokens over a paged cache: one token of each request, a tree of drafted ones, or a causal chunk.
//
//   token j of request b sees the cached keys [0, p), p = kv_len - n, and of the n new ones, which the cache holds as
//   well, those that its mask names (no masks: 0 .. j);   o = sum_key softmax(scale q.key) value
//
// One pass over the keys with the running maximum and sum of the softmax, both fp32, as is the output until its one
// rounding.  A token that sees nothing gives 0 and -inf.
//
// With a window W and S first tokens (LOCAL kernels): the keys that a token may see as above, numbered from 0 in the cache's order, of
// which it sees the last W and the first S.
#pragma once
#include <math.h>
#include <type_traits>
#include "moe_common.h"
#include "moe_layout.h"
#include "attn_reach.h"
#include "lanes.h"
#include "../../include/moe_hip.h"

namespace moe {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

struct AttnArgs {
  const uint16_t *q;
  int64_t q_stride;
  int T, Hq, Hkv, G, B, n_blocks, page_log2, table_width;
  const uint8_t *k_cache, *v_cache;
  uint32_t k_block_bytes, v_block_bytes;
  int64_t table_stride;
  const int32_t *tables, *kv_lens, *cu;
  const int64_t *masks;
  float scale;
  const float *k_scale, *v_scale;
  uint16_t *out;
  float *lse;
  int groups;                          // workgroups of the main launch
  float cut;                           // see attn_walk
  float *part_o, *part_ml;             // [2 groups][rows][D]; [2 groups][rows][2]
  int32_t *records;                    // [groups][8]: of the tile that begins in a stretch and goes on: last stretch, the
                                       // request's first row and rows, head, tile, part
  uint32_t most_units;                 // the line's length at most
  // LOCAL kernels: window and first tokens; of a cache in 4 bits the powers of two, a byte to 32 elements
  int window, sinks;
  const uint8_t *k_powers, *v_powers;  // [n_blocks][page][Hkv][D / 32]
  uint32_t k_powers_block, v_powers_block;
};

// ---- who does what ----------------------------------------------------------------------------------------------------
// The work is a line of units: for each request, each cache head, each tile of ROWS of its rows (a row: a token and a query
// head of the cache head's group), each UNIT keys that the tile sees.  Every workgroup takes an equal stretch of the line,
// which may begin and end inside a tile and hold several, so that ragged lengths cost nothing.  A tile that lies in one stretch
// is finished there; of the others each stretch leaves (max, sum, weighted values), which the second launch joins in
// order.
struct AttnRequest {
  int t0, n, kv, prefix;
};
__device__ __forceinline__ AttnRequest attn_request(const AttnArgs &a, int b) {
  const int t0 = min(max(a.cu[b], 0), a.T), t1 = min(max(a.cu[b + 1], t0), a.T);
  const int kv = (int)min((int64_t)a.kv_lens[b], (int64_t)a.table_width << a.page_log2);
  return {t0, t1 - t0, kv, kv - (t1 - t0)};
}
template <int ROWS, int UNIT, bool LOCAL>
__device__ __forceinline__ AttnReach attn_reach(const AttnArgs &a, const AttnRequest &r, int m) {
  if (LOCAL) return attn_window_reach(ROWS, UNIT, a.masks, r.n, a.G, r.prefix, r.kv, a.window, a.sinks, m);
  return {(attn_tile_end(ROWS, a.masks, r.n, a.G, r.prefix, r.kv, m) + UNIT - 1) / UNIT, 0, 0, 0, 0, 0};
}
template <int ROWS, int UNIT>
__device__ __forceinline__ int attn_head_units(const AttnArgs &a, const AttnRequest &r) {
  if (r.n <= 0 || r.prefix < 0) return 0;
  const int tiles = (r.n * a.G + ROWS - 1) / ROWS;
  if (a.masks || r.n == 1) return tiles * attn_reach<ROWS, UNIT, false>(a, r, 0).units;
  int sum = 0;
  for (int m = 0; m < tiles; m++) sum += attn_reach<ROWS, UNIT, false>(a, r, m).units;
  return sum;
}

// A workgroup's way along its stretch: calls segment(request, head, tile, units c0 .. c1 of the tile's u, part) for each piece.
// Every wavefront adds the line up for itself, 64 requests at a time, and finds its first request among them: one trip to
// memory and no barrier stand in front of the work.  The host has seen to it that the line's length fits an int where cu_tokens ascends;
// where it does not, requests share rows and the line may have any length: a longer one than the host allowed for is taken for empty, so that
// no index wraps and every walk ends.
template <int ROWS, int UNIT, typename Segment>
__device__ __forceinline__ void attn_walk(const AttnArgs &a, Segment segment) {
  const int lane = threadIdx.x & 63;
  AttnRequest mine{0, 0, 0, -1};
  int units = 0, longest = 0;
  uint32_t upto = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    if (b0 + lane < a.B) mine = attn_request(a, b0 + lane);
    else mine.n = 0;
    units = attn_head_units<ROWS, UNIT>(a, mine) * a.Hkv;
    upto = __builtin_elementwise_add_sat(upto, (uint32_t)units);
    if (units > 0) longest = max(longest, (mine.kv + UNIT - 1) / UNIT);
  }
  upto = lane_sum_upto(upto);                          // (with up to 64 requests: the line's length up to each)
  int total = __builtin_amdgcn_readlane(upto, 63);
  if ((uint32_t)total > a.most_units) total = 0;
  longest = __builtin_amdgcn_readfirstlane(lane_max(longest));
  // An equal share for every workgroup, but of one long tile no more than pays: n units cut into stretches of x take x steps of a unit, then
  // a join of n / x parts, least at x = sqrt(n cut), cut the time of a part over that of a unit.  (One token over 32767 keys: 28, 23.5 and
  // 26 us with stretches of 2, 4 and 8 units; over 1000 keys 14.8 and 17.8 us with 2 and 4.)
  const int even = (int)(((uint32_t)total + a.groups - 1) / (uint32_t)a.groups), least = __builtin_amdgcn_readfirstlane((int)ceilf(sqrtf((float)longest * a.cut)));
  const int per = max(max(even, least), 1);
  // Neighbouring stretches, whose tiles have keys in common, on one XCD and so behind one L2: workgroups go to the eight XCDs in turn.
  const int eighth = (int)(((uint32_t)total + per - 1) / (uint32_t)per + 7) / 8, wg = blockIdx.x, place = wg < 8 * eighth ? wg % 8 * eighth + wg / 8 : wg;
  const int start = (int)min((int64_t)place * per, (int64_t)total), end = start + min(per, total - start);
  if (threadIdx.x == 0) a.records[8 * place] = -1;
  if (start >= end) return;
  int b = 0, before = 0;
  AttnRequest r{};
  for (int b0 = 0;; b0 += 64) {                        // (ends: start < total)
    if (a.B > 64) {
      if (b0 + lane < a.B) mine = attn_request(a, b0 + lane);
      else mine.n = 0;
      units = attn_head_units<ROWS, UNIT>(a, mine) * a.Hkv;
      upto = lane_sum_upto(units);
    }
    const uint64_t past = __ballot(start < before + (int)upto);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      before += __builtin_amdgcn_readlane((int)upto - units, l);
      r = {__builtin_amdgcn_readlane(mine.t0, l), __builtin_amdgcn_readlane(mine.n, l), __builtin_amdgcn_readlane(mine.kv, l),
           __builtin_amdgcn_readlane(mine.prefix, l)};
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  for (int at = start;;) {
    const int head = attn_head_units<ROWS, UNIT>(a, r);
    if (at >= before + head * a.Hkv) {
      before += head * a.Hkv;
      r = attn_request(a, ++b);
      continue;
    }
    const int kh = (at - before) / head, in_head = at - before - kh * head;
    int m = 0, u = (r.kv + UNIT - 1) / UNIT, first = 0;
    if (a.masks || r.n == 1) {
      m = in_head / u;
      first = m * u;
    } else {
      for (;; m++) {
        u = attn_reach<ROWS, UNIT, false>(a, r, m).units;
        if (in_head < first + u) break;
        first += u;
      }
    }
    const int c0 = in_head - first, c1 = min(u, c0 + (end - at));
    if (threadIdx.x == 0 && c0 == 0 && c1 < u) {
      int32_t *rec = a.records + 8 * place;
      rec[0] = (at + u - 1) / per, rec[1] = r.t0, rec[2] = r.n, rec[3] = kh, rec[4] = m, rec[5] = at > start;
    }
    segment(r, b, kh, m, c0, c1, c0 == 0 && c1 == u, 2 * place + (at - c0 > start ? 1 : 0));
    at += c1 - c0;
    if (at >= end) break;
  }
}

// The same for LOCAL kernels.  With a window most tiles are equally long, and lengths may be alike without one: where all tiles filled up to the longest
// one's length are not more than an eighth longer, the line has every tile at that length, and stretches are whole tiles or a tile's equal parts, so that
// none holds the end of one tile and the beginning of the next and, of whole tiles, nothing is left to join (two chunks of 1021 tokens
// in a window of 1024, 32 query heads: 84 us with stretches across tiles, 59 so).  A lane adds up
// a tile of a causal request, 64 at once.
template <int ROWS, int UNIT, int HEADS, typename Segment>
__device__ __forceinline__ void attn_walk_local(const AttnArgs &a, Segment segment) {
  const int lane = threadIdx.x & 63, heads = a.Hkv / HEADS;
  const auto tiles_of = [&](const AttnRequest &r) { return r.n <= 0 || r.prefix < 0 ? 0 : (r.n * a.G + ROWS - 1) / ROWS; };
  const auto alike = [&](const AttnRequest &r) { return a.masks || r.n == 1; };        // all tiles of the request
  struct Tiles {
    int units, longest;                // of all tiles of a request for a head; of the longest of them
  };
  // of a request that all lanes hold, a tile to a lane
  const auto sum_of = [&](const AttnRequest &r) {
    const int tiles = tiles_of(r);
    if (alike(r)) {
      const int u = tiles ? attn_reach<ROWS, UNIT, true>(a, r, 0).units : 0;
      return Tiles{tiles * u, u};
    }
    int sum = 0, most = 0;
    for (int m = 0; m < tiles; m += 64) {
      const int u = m + lane < tiles ? attn_reach<ROWS, UNIT, true>(a, r, m + lane).units : 0;
      sum += __builtin_amdgcn_readlane(lane_sum_upto((uint32_t)u), 63);
      most = max(most, u);
    }
    return Tiles{sum, __builtin_amdgcn_readfirstlane(lane_max(most))};
  };
  const auto of_lane = [&](const AttnRequest &r, int l) {
    return AttnRequest{__builtin_amdgcn_readlane(r.t0, l), __builtin_amdgcn_readlane(r.n, l), __builtin_amdgcn_readlane(r.kv, l), __builtin_amdgcn_readlane(r.prefix, l)};
  };
  // of 64 requests, one to a lane: the units of each one's tiles (a lane by itself, or all of them for one request after the other if that
  // takes fewer turns)
  const auto head_units = [&](const AttnRequest &r) {
    const int tiles = tiles_of(r), turns = alike(r) ? 1 : tiles;
    const int most = __builtin_amdgcn_readfirstlane(lane_max(turns)), together = __builtin_amdgcn_readlane(lane_sum_upto((uint32_t)(turns + 63) / 64), 63);
    Tiles t{0, 0};
    if (most <= 2 * together) {
      if (alike(r)) {
        t.longest = tiles ? attn_reach<ROWS, UNIT, true>(a, r, 0).units : 0;
        t.units = tiles * t.longest;
      } else {
        for (int m = 0; m < tiles; m++) {
          const int u = attn_reach<ROWS, UNIT, true>(a, r, m).units;
          t.units += u;
          t.longest = max(t.longest, u);
        }
      }
      return t;
    }
    for (uint64_t todo = __ballot(tiles > 0); todo; todo &= todo - 1) {
      const int l = __builtin_ctzll(todo);
      const Tiles its = sum_of(of_lane(r, l));
      if (lane == l) t = its;
    }
    return t;
  };
  const auto request = [&](int b) { return b < a.B ? attn_request(a, b) : AttnRequest{0, 0, 0, -1}; };

  AttnRequest mine{0, 0, 0, -1};
  int units = 0, longest = 0;
  uint32_t upto = 0, tiles = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    mine = request(b0 + lane);
    const Tiles its = head_units(mine);
    units = its.units * heads;
    longest = max(longest, its.longest);
    upto = __builtin_elementwise_add_sat(upto, (uint32_t)units);
    tiles = __builtin_elementwise_add_sat(tiles, (uint32_t)(tiles_of(mine) * heads));
  }
  upto = lane_sum_upto(upto);                          // (with up to 64 requests: the line's length up to each)
  int total = __builtin_amdgcn_readlane(upto, 63);
  if ((uint32_t)total > a.most_units) total = 0;
  tiles = __builtin_amdgcn_readlane(lane_sum_upto(tiles), 63);
  longest = __builtin_amdgcn_readfirstlane(lane_max(longest));
  const int even = (int)(((uint32_t)total + a.groups - 1) / (uint32_t)a.groups), least = max(__builtin_amdgcn_readfirstlane((int)ceilf(sqrtf((float)longest * a.cut))), 1);
  int per = max(max(even, least), 1), filled = 0;      // filled: the length of every tile on the line, or 0: their own
  if (total > 0 && (uint64_t)tiles * (uint64_t)longest * 8 <= (uint64_t)total * 9) {
    const uint32_t groups = (uint32_t)a.groups;
    if (tiles >= groups) {                             // some tiles to each workgroup, if few of these go without
      const uint32_t each = (tiles + groups - 1) / groups;
      if ((uint64_t)tiles * 8 >= (uint64_t)groups * each * 7) filled = longest, per = longest * (int)each;
    } else {                                           // a tile to some workgroups
      const int share = (int)(groups / tiles), most = max(longest / least, 1), pieces = min(share, most);
      if (most < share || tiles * (uint32_t)pieces * 8 >= groups * 7) {
        per = (longest + pieces - 1) / pieces;
        filled = per * ((longest + per - 1) / per);
      }
    }
    if ((uint64_t)tiles * (uint64_t)filled > 0x7fffffffull) filled = 0, per = max(even, least);
  }
  if (filled) {
    total = (int)tiles * filled;
    units = tiles_of(mine) * heads * filled;
    upto = lane_sum_upto((uint32_t)units);
  }
  // Neighbouring stretches on one XCD, as above.
  const int eighth = (int)(((uint32_t)total + per - 1) / (uint32_t)per + 7) / 8, wg = blockIdx.x, place = wg < 8 * eighth ? wg % 8 * eighth + wg / 8 : wg;
  const int start = (int)min((int64_t)place * per, (int64_t)total), end = start + min(per, total - start);
  if (threadIdx.x == 0) a.records[8 * place] = -1;
  if (start >= end) return;
  int b = 0, before = 0;
  AttnRequest r{};
  for (int b0 = 0;; b0 += 64) {                        // (ends: start < total)
    if (a.B > 64) {
      mine = request(b0 + lane);
      units = filled ? tiles_of(mine) * heads * filled : head_units(mine).units * heads;
      upto = lane_sum_upto((uint32_t)units);
    }
    const uint64_t past = __ballot(start < before + (int)upto);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      before += __builtin_amdgcn_readlane((int)upto - units, l);
      r = of_lane(mine, l);
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  int head = filled ? tiles_of(r) * filled : sum_of(r).units;
  for (int at = start;;) {
    if (at >= before + head * heads) {
      before += head * heads;
      r = attn_request(a, ++b);
      head = filled ? tiles_of(r) * filled : sum_of(r).units;
      continue;
    }
    const int kh = (at - before) / head, in_head = at - before - kh * head;
    int m = 0, u = 0, slots = filled, first = 0;
    if (filled || alike(r)) {
      if (!filled) slots = attn_reach<ROWS, UNIT, true>(a, r, 0).units;
      m = in_head / slots;
      first = m * slots;
      u = attn_reach<ROWS, UNIT, true>(a, r, m).units;
    } else {
      for (;; m += 64) {                               // (ends: the tiles' units add up to more than in_head)
        const int own = m + lane < tiles_of(r) ? attn_reach<ROWS, UNIT, true>(a, r, m + lane).units : 0;
        const int so_far = first + (int)lane_sum_upto((uint32_t)own);
        const uint64_t past = __ballot(in_head < so_far);
        if (past) {
          const int l = __builtin_ctzll(past);
          m += l;
          u = slots = __builtin_amdgcn_readlane(own, l);
          first = __builtin_amdgcn_readlane(so_far, l) - u;
          break;
        }
        first = __builtin_amdgcn_readlane(so_far, 63);
      }
    }
    const int c0 = in_head - first, c1 = min(u, c0 + (end - at));
    if (c0 < u) {                                      // (behind it the tile is filled up)
      if (threadIdx.x == 0 && c0 == 0 && c1 < u) {
        int32_t *rec = a.records + 8 * place;
        rec[0] = (at + u - 1) / per, rec[1] = r.t0, rec[2] = r.n, rec[3] = kh, rec[4] = m, rec[5] = at > start;
      }
      segment(r, b, kh, m, c0, c1, c0 == 0 && c1 == u, 2 * place + (at - c0 > start ? 1 : 0));
    }
    at += min(slots - c0, end - at);
    if (at >= end) break;
  }
}
// LOCAL or not
template <int ROWS, int UNIT, bool LOCAL, int HEADS, typename Segment>
__device__ __forceinline__ void attn_go(const AttnArgs &a, Segment segment) {
  if constexpr (LOCAL) attn_walk_local<ROWS, UNIT, HEADS>(a, segment);
  else attn_walk<ROWS, UNIT>(a, segment);
}

// ---- softmax and products of 32 keys ----------------------------------------------------------------------------------
// Scores are formed transposed, S^T = K Q^T, so that a lane holds for ONE query (lane % 16) the keys 4 g + i, g = lane / 16, of two
// tiles of 16.  Those eight are at once the lane's operand of O^T = V^T P^T, if the reduction runs over the keys in that
// order: no probability changes its lane.  V^T comes from row-major values in LDS by the transposing read.
// p = 2^(s c - m): m lies kLag above the maximum of a tile's first keys and follows it later only where a lane's probabilities add up to more than 1, so
// that in between no maximum is formed nor anything rescaled.  The largest p is between about 2^-kLag and 1: sums of p v are no larger
// than the softmax's own before its division, and they lose what is smaller than 2^(kLag - 126).  p is rounded to bf16 for the product (what
// the matrix cores take; an error of 2^-9 of each term, as the output's own rounding); its sum is taken before that, in fp32.
constexpr float kLag = 16.f;                           // (scores that outgrow the first keys' by 11 raise m, a few times a tile at the most)
__device__ __forceinline__ float over_groups(float v, bool sum) {
  v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = sum ? __uint_as_float(r[0]) + __uint_as_float(r[1]) : fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum ? __uint_as_float(r[0]) + __uint_as_float(r[1]) : fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int NQ, int DT>
struct AttnState {
  v4f o[DT][NQ];
  float m[NQ], l[NQ];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) {
      m[qc] = -INFINITY;
      l[qc] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; dt++) o[dt][qc] = (v4f){0.f, 0.f, 0.f, 0.f};
    }
  }
  // lets m follow the largest of KT tiles' scores (a little more is left alone)
  template <int KT>
  __device__ __forceinline__ void raise(const v4f (&s)[KT][NQ], float c) {
    float top[NQ];
    bool grown = false;
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) {
      float t = s[0][qc][0];
#pragma unroll
      for (int x = 1; x + 1 < 4 * KT; x += 2) t = fmaxf(fmaxf(t, s[x / 4][qc][x % 4]), s[(x + 1) / 4][qc][(x + 1) % 4]);
      top[qc] = fmaxf(t, s[KT - 1][qc][3]) * c;
      grown |= top[qc] > m[qc] + 8.f;
    }
    if (__builtin_expect(__any(grown), 0)) {
#pragma unroll
      for (int qc = 0; qc < NQ; qc++) {
        const float t = over_groups(top[qc], false), now = t > m[qc] - kLag + 8.f ? t + kLag : m[qc];
        const float f = now == m[qc] ? 1.f : __builtin_amdgcn_exp2f(m[qc] - now);
        m[qc] = now;
        l[qc] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt][qc] *= f;
      }
    }
  }
  // KT tiles' scores -> probabilities, as the second product's operands.  sure: m follows the maximum first (a tile's first
  // keys, and keys that some rows do not see); else m is left alone unless the sums show that it is far too low.
  template <int KT>
  __device__ __forceinline__ void softmax(const v4f (&s)[KT][NQ], float c, bool sure, v8bf (&p)[KT / 2][NQ]) {
    float sum[NQ];
    for (bool rise = sure;;) {
      if (__builtin_expect(rise, 0)) raise<KT>(s, c);
      weigh<KT>(s, c, p, sum);
      bool far = false;
#pragma unroll
      for (int qc = 0; qc < NQ; qc++) far |= sum[qc] > 1.f;
      if (__builtin_expect(rise || !__any(far), 1)) break;
      rise = true;
    }
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) l[qc] += sum[qc];
  }
  template <int KT>
  __device__ __forceinline__ void weigh(const v4f (&s)[KT][NQ], float c, v8bf (&p)[KT / 2][NQ], float (&sum)[NQ]) const {
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) {
      sum[qc] = 0.f;
      const float off = m[qc] == -INFINITY ? 0.f : m[qc];
#pragma unroll
      for (int h = 0; h < KT / 2; h++) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = __builtin_amdgcn_exp2f(fmaf(s[2 * h + i / 4][qc][i % 4], c, -off));
        sum[qc] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        const v4i w = {(int)pack2_bf16(e[0], e[1]), (int)pack2_bf16(e[2], e[3]), (int)pack2_bf16(e[4], e[5]), (int)pack2_bf16(e[6], e[7])};
        p[h][qc] = __builtin_bit_cast(v8bf, w);
      }
    }
  }
};

// The products' operands come from LDS some hundred cycles after they are asked for, a group of matrix instructions takes 32 to 64: operands
// are asked for AHEAD groups before their use, and the order written here is kept (left to itself the compiler asks
// and waits in turn: 683 instead of 728 TFLOP/s with 2042 rows of a chunk over 8190 keys).
__device__ __forceinline__ void in_this_order() { __builtin_amdgcn_sched_barrier(0); }
__device__ __forceinline__ void made_here(v4f &x) { asm volatile("" : "+v"(x)); }      // (products are moved freely otherwise)

// 16 columns of the values of 32 keys as the product's first operand; `at`: this lane's address in the first 16 rows
template <int LD>
__device__ __forceinline__ v8bf attn_values(const uint8_t *at, int dt) {
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(at + 32 * dt));
  const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(at + 16 * LD + 32 * dt));
  return __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// o += V^T p over H times 32 keys; v: the first AHEAD operands, asked for already
template <int AHEAD, int H, int LD, int NQ, int DT>
__device__ __forceinline__ void attn_add_values(AttnState<NQ, DT> &st, const uint8_t *at, const v8bf (&p)[H][NQ], v8bf (&v)[H * DT]) {
#pragma unroll
  for (int i = 0; i < H * DT; i++) {
    if (i + AHEAD < H * DT) v[i + AHEAD] = attn_values<LD>(at + 32 * ((i + AHEAD) / DT) * LD, (i + AHEAD) % DT);
    in_this_order();
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) {
      st.o[i % DT][qc] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[i], p[i / DT][qc], st.o[i % DT][qc], 0, 0, 0);
      made_here(st.o[i % DT][qc]);
    }
    in_this_order();
  }
}
// scores of KT tiles of 16 keys, rows LK apart in LDS from `at` (this lane's row of the first tile and its 16 bytes) on
template <int AHEAD, int KT, int LK, int NQ, int X>
__device__ __forceinline__ void attn_scores(const uint8_t *at, const v8bf (&q)[NQ][X], v4f (&s)[KT][NQ]) {
  v8bf k[KT * X];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) k[i] = *(const v8bf *)(at + (i / X) * 16 * LK + 64 * (i % X));
#pragma unroll
  for (int i = 0; i < KT * X; i++) {
    if (i + AHEAD < KT * X) k[i + AHEAD] = *(const v8bf *)(at + ((i + AHEAD) / X) * 16 * LK + 64 * ((i + AHEAD) % X));
    in_this_order();
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) {
      s[i / X][qc] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[i], q[qc][i % X], i % X ? s[i / X][qc] : (v4f){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      made_here(s[i / X][qc]);
    }
    in_this_order();
  }
}

// what a lane's queries see of the new tokens
__device__ __forceinline__ uint64_t attn_first(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }
template <int NQ, bool LOCAL>
struct AttnSight {
  uint64_t mask[NQ];                   // without masks: the last key seen
  int lowest[LOCAL ? NQ : 1];          // the first cached key in the window
  // bit k: query qc sees key first_key + k
  __device__ __forceinline__ uint64_t from(const AttnArgs &a, const AttnRequest &r, int qc, int first_key) const {
    const uint64_t near = LOCAL ? ~attn_first(lowest[LOCAL ? qc : 0] - first_key) | attn_first(a.sinks - first_key) : ~0ull;
    if (!a.masks) return near & attn_first((int)mask[qc] + 1 - first_key);
    const int i = first_key - r.prefix;                // the first key's bit
    return near & attn_first(r.kv - first_key) & (i >= 64 ? 0ull : i >= 0 ? mask[qc] >> i : i > -64 ? mask[qc] << -i | attn_first(-i) : ~0ull);
  }
  // the row of token j, which may see the new tokens of `may`
  __device__ __forceinline__ void set(const AttnArgs &a, const AttnRequest &r, int qc, int j, uint64_t may) {
    mask[qc] = a.masks ? may : (uint64_t)(r.prefix + j);
    if (!LOCAL) return;
    if (!a.masks) {
      lowest[LOCAL ? qc : 0] = max(r.prefix + j + 1 - a.window, 0);
      return;
    }
    may &= attn_first(r.n);
    const int count = __popcll(may), head = min(max(a.sinks - r.prefix, 0), count);
    lowest[LOCAL ? qc : 0] = max(min(r.prefix + count - a.window, r.prefix), 0);
    int drop = count - a.window - head;                // new tokens that lie between the first ones and the window
    if (drop > 0) {
      uint64_t kept = 0;
      for (int i = 0; i < head; i++) kept |= may & -may, may &= may - 1;
      for (; drop > 0; drop--) may &= may - 1;
      may |= kept;
    }
    mask[qc] = may;
  }
};

// Hides what a lane's queries do not see; the scores left are scaled already.
template <int NQ, bool LOCAL, int KT>
__device__ __forceinline__ void attn_hide(const AttnArgs &a, const AttnRequest &r, const AttnSight<NQ, LOCAL> &sight, int first_key, float c,
                                          v4f (&s)[KT][NQ]) {
  const int g4 = 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int qc = 0; qc < NQ; qc++) {
    const uint64_t seen = sight.from(a, r, qc, first_key) >> g4;
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int i = 0; i < 4; i++) s[kt][qc][i] = seen >> (16 * kt + i) & 1 ? s[kt][qc][i] * c : -INFINITY;
  }
}

// What a lane holds of a key or value, and how it becomes operands of 8 bf16: BYTES bytes are E elements.
//   bf16, e4m3    16 bytes: themselves, or two operands of e4m3 codes
//   4 bits        16 bytes: four operands, or 8 bytes: two; codes of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives times a power of two, which
//                 bf16 holds exactly, so that the conversion that applies the power rounds nothing
template <int C, int B = 16>
struct AttnPiece {
  static constexpr int BYTES = B, E = C == MOE_DTYPE_BF16 ? B / 2 : C == MOE_DTYPE_FP8 ? B : 2 * B;
  uint32_t w[B / 4];
  __device__ __forceinline__ void load(const uint8_t *at) {
    if constexpr (B == 16) {
      const v4i v = *(const v4i *)at;
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = (uint32_t)v[i];
    } else {
      const v2i v = *(const v2i *)at;
#pragma unroll
      for (int i = 0; i < 2; i++) w[i] = (uint32_t)v[i];
    }
  }
  __device__ __forceinline__ v8bf operand(int h, float power) const {
    v4i r;
    if constexpr (C == MOE_DTYPE_BF16) {
      r = (v4i){(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    } else if constexpr (C == MOE_DTYPE_FP8) {
      const uint32_t w0 = w[2 * h], w1 = w[2 * h + 1];
      r = (v4i){__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true))};
    } else {
      r = (v4i){__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[h], power, 0)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[h], power, 1)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[h], power, 2)),
                __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[h], power, 3))};
    }
    return __builtin_bit_cast(v8bf, r);
  }
};
constexpr int attn_row_bytes(int C, int D) { return C == MOE_DTYPE_BF16 ? 2 * D : C == MOE_DTYPE_FP8 ? D : D / 2; }
// two bf16 in a word: which are NaN or infinite -> 0xffff in their place
__device__ __forceinline__ uint32_t no_numbers(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

__device__ __forceinline__ int attn_block(const AttnArgs &a, const int32_t *table, int key) {
  return min(max(table[key >> a.page_log2], 0), a.n_blocks - 1);
}
// where a head's key or value of a block lies (one 32 x 32 -> 64 bit multiplication and one of 24 bits)
template <int BYTES>
__device__ __forceinline__ const uint8_t *attn_row(const AttnArgs &a, const uint8_t *cache, uint32_t block_bytes, int block, int kh, int key) {
  return cache + (uint64_t)(uint32_t)block * block_bytes +
         (__umul24((uint32_t)key & ((1u << a.page_log2) - 1), (uint32_t)a.Hkv * BYTES) + (uint32_t)kh * BYTES);
}
// the power of two of element d of a key or value in 4 bits: a byte, the exponent of a float
template <int D>
__device__ __forceinline__ uint32_t attn_power(const AttnArgs &a, const uint8_t *powers, uint32_t block_bytes, int block, int kh, int key, int d) {
  return attn_row<D / 32>(a, powers, block_bytes, block, kh, key)[d / 32];
}
__device__ __forceinline__ float attn_power_value(uint32_t byte) { return __uint_as_float(byte << 23); }

// A value that is NaN or infinite would, times a probability of 0, reach rows that do not see its key.  Where new tokens are among
// the keys such values are staged as 0, and this adds them to the rows that do see them.
template <int NQ, int DT, int C, bool LOCAL>
__device__ __forceinline__ void attn_add_no_numbers(const AttnArgs &a, const AttnRequest &r, const AttnSight<NQ, LOCAL> &sight, const int32_t *table,
                                                 int kh, int first_key, int keys, AttnState<NQ, DT> &st) {
  const int g4 = 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll 1
  for (int key = first_key; key < min(first_key + keys, r.kv); key++) {
    if (LOCAL) {                                       // (a page that no row sees may not be the request's any more)
      bool some = false;
#pragma unroll
      for (int qc = 0; qc < NQ; qc++) some |= sight.from(a, r, qc, key) & 1;
      if (!__any(some)) continue;
    }
    const int block = attn_block(a, table, key);
    const uint8_t *row = attn_row<attn_row_bytes(C, 16 * DT)>(a, a.v_cache, a.v_block_bytes, block, kh, key);
    bool sees[NQ];
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) sees[qc] = sight.from(a, r, qc, key) & 1;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int d = 16 * dt + g4 + i;
        float v;
        if constexpr (C == MOE_DTYPE_BF16) {
          v = bf16_to_f32(((const uint16_t *)row)[d]);
        } else if constexpr (C == MOE_DTYPE_FP8) {
          v = __builtin_amdgcn_cvt_f32_fp8((uint32_t)row[d], 0);
        } else {
          const float power = attn_power_value(attn_power<16 * DT>(a, a.v_powers, a.v_powers_block, block, kh, key, d));
          const uint32_t two = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)row[d / 2], power, 0));
          v = bf16_to_f32((uint16_t)(d & 1 ? two >> 16 : two));
        }
        v = __builtin_isfinite(v) ? 0.f : v;
#pragma unroll
        for (int qc = 0; qc < NQ; qc++) st.o[dt][qc][i] += sees[qc] ? v : 0.f;
      }
  }
}

// a lane's queries as the scores' second operand: element j of step s is d = 32 s + 8 g + j, or where a lane reads E > 8 neighbouring elements
// of a key (16 in e4m3, D / 4 in 4 bits) in the order of its keys, d = 4 E (s / (E / 8)) + E g + 8 (s % (E / 8)) + j.  Its 16s of rows lie STEP apart.  Of the scores' factor the queries take the
// sign, so that the largest score is the largest product.
template <int NQ, int D, int E, bool LOCAL, int STEP = 16>
__device__ __forceinline__ void attn_queries(const AttnArgs &a, const AttnRequest &r, int kh, int first_row, float factor, v8bf (&q)[NQ][D / 32],
                                             AttnSight<NQ, LOCAL> &sight) {
  const int lane = threadIdx.x & 63, g = lane >> 4, flip = factor < 0.f ? (int)0x80008000 : 0;
#pragma unroll
  for (int qc = 0; qc < NQ; qc++) {
    const int row = min(first_row + STEP * qc + (lane & 15), r.n * a.G - 1), j = row / a.G, h = kh * a.G + row - j * a.G;
    const uint16_t *src = a.q + (size_t)(r.t0 + j) * a.q_stride + (size_t)h * D;
#pragma unroll
    for (int s = 0; s < D / 32; s++) {
      const v4i w = *(const v4i *)(src + 4 * E * (s / (E / 8)) + E * g + 8 * (s % (E / 8)));
      q[qc][s] = __builtin_bit_cast(v8bf, w ^ flip);
    }
    sight.set(a, r, qc, j, a.masks ? (uint64_t)a.masks[r.t0 + j] : 0);
  }
}

// Four neighbouring outputs of a row: finished, or as a stretch's part of it.
template <int ROWS, int D>
__device__ __forceinline__ void attn_store(const AttnArgs &a, const AttnRequest &r, int kh, int m_tile, int row_in_tile, int d, bool whole,
                                           int part, const v4f o, float m, float l) {
  const int row = m_tile * ROWS + row_in_tile;
  if (row >= r.n * a.G) return;
  if (!whole) {
    *(v4f *)(a.part_o + ((size_t)part * ROWS + row_in_tile) * D + d) = o;
    if (d == 0) {
      a.part_ml[((size_t)part * ROWS + row_in_tile) * 2] = m;
      a.part_ml[((size_t)part * ROWS + row_in_tile) * 2 + 1] = l;
    }
    return;
  }
  const int j = row / a.G, h = kh * a.G + row - j * a.G;
  const size_t at = (size_t)(r.t0 + j) * a.Hq + h;
  const bool none = m == -INFINITY && l == 0.f;
  const float f = none ? 0.f : (a.v_scale ? a.v_scale[kh] : 1.f) / l;
  *(v2i *)(a.out + at * D + d) = (v2i){(int)pack2_bf16(o[0] * f, o[1] * f), (int)pack2_bf16(o[2] * f, o[3] * f)};
  if (a.lse && d == 0) a.lse[at] = none ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// ---- few rows: the four wavefronts take the keys in turn --------------------------------------------------------------
// Up to 16 rows to a cached key the cache's bytes bound it (64 requests, up to 8192 keys, bf16: 134 us, 4.9 TB/s, what a large copy reaches;
// one request of 32767: 23.4 us, of which 14 are its bytes and the rest the chain of launch, lengths, tables, a tile's end and the join).  A wavefront takes 32 keys of a unit of 128 by itself: keys go
// from memory straight into operand registers, values through LDS that no other wavefront touches, so nothing waits at a
// barrier, and the next keys and values are asked for before the present ones are worked on.  The wavefronts' results meet in
// LDS at the end of a tile.
// In 4 bits a head's key is 64 bytes or 32, half a line of memory or less, so that one head's keys alone come at 2.6 to 2.9 TB/s.  With HEADS = 2 a
// workgroup reads two neighbouring heads' keys at the same time, a pair of wavefronts (SHARE) to each: 4.0 TB/s (256 requests of up to 8192 keys, 4 heads: 261 us with
// one head, 174 with two; e4m3 heads of 64: 462 and 269 over 8 heads, 4.9 TB/s).  (Four heads: 246 us where two take 294, 256 requests of 8 heads of
// 64 in 4 bits; no faster elsewhere, slower where parts have to be joined.)
template <int D, int C, bool LOCAL, int NQ, int HEADS>
__global__ __launch_bounds__(256, 2) void attn_keys_kernel(const AttnArgs a) {
  constexpr int ROWS = 16 * NQ, SHARE = 4 / HEADS, UNIT = 32 * SHARE, DT = D / 16, LD = 2 * D + 32;
  using Piece = AttnPiece<C, C == MOE_DTYPE_FP4 ? D / 8 : 16>;
  constexpr int E = Piece::E, P = D / (4 * E);         // a lane's pieces of a key
  constexpr int kValues = 4 * 32 * LD, kMerge = 4 * DT * NQ * 64 * 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kValues > kMerge ? kValues : kMerge];
  __shared__ float sh_m[4][ROWS], sh_l[4][ROWS];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
  const int of_head = w % HEADS, part_of_unit = w / HEADS;
  uint8_t *values = lds + w * 32 * LD;
  const uint8_t *read_at = values + (4 * g + c16 / 4) * LD + 8 * (c16 % 4);
  attn_go<ROWS, UNIT, LOCAL, HEADS>(a, [&](const AttnRequest r, int b, int first_head, int m_tile, int c0, int c1, bool whole, int part) {
    const int kh = first_head * HEADS + of_head;
    const int32_t *table = a.tables + (size_t)b * a.table_stride;
    const float factor = a.scale * (a.k_scale ? a.k_scale[kh] : 1.f) * 1.4426950408889634f, scale = fabsf(factor);
    v8bf q[NQ][D / 32];
    AttnSight<NQ, LOCAL> sight;
    attn_queries<NQ, D, E>(a, r, kh, m_tile * ROWS, factor, q, sight);
    const int clear = a.masks ? r.prefix : r.prefix + m_tile * ROWS / a.G + 1;      // keys below it are seen by every row
    const AttnReach reach = attn_reach<ROWS, UNIT, LOCAL>(a, r, m_tile);            // (and from reach.every on)
    AttnState<NQ, DT> st;
    st.clear();
    // The block of a key is read two units ahead of the key, so that no load waits for another one.
    Piece kr[2][P], vr[2][P];
    uint32_t kp[2], vp[2];                             // their powers of two
    int block[2];
    const auto key_of = [&](int unit, int kt) {
      const int key = reach.unit(unit) * UNIT + 32 * part_of_unit + 16 * kt + c16;
      return min(LOCAL ? reach.read(key) : key, r.kv - 1);
    };
    const auto blocks = [&](int unit) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++) block[kt] = attn_block(a, table, key_of(unit, kt));
    };
    const auto load = [&](bool values, int unit, Piece (&to)[2][P], uint32_t (&powers)[2]) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++) {
        const int key = key_of(unit, kt);
        const uint8_t *row = attn_row<attn_row_bytes(C, D)>(a, values ? a.v_cache : a.k_cache, values ? a.v_block_bytes : a.k_block_bytes, block[kt], kh, key) +
                             Piece::BYTES * g;
#pragma unroll
        for (int p = 0; p < P; p++) to[kt][p].load(row + 4 * Piece::BYTES * p);
        if (C == MOE_DTYPE_FP4)
          powers[kt] = attn_power<D>(a, values ? a.v_powers : a.k_powers, values ? a.v_powers_block : a.k_powers_block, block[kt], kh, key, E * g);
      }
    };
    blocks(c0);
    load(false, c0, kr, kp);
    load(true, c0, vr, vp);
    bool sure = true;                                  // the next keys may be the first that a row sees
    blocks(min(c0 + 1, c1 - 1));
    for (int c = c0; c < c1; c++) {
      const int key0 = reach.unit(c) * UNIT + 32 * part_of_unit;
      v4f s[2][NQ];
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int qc = 0; qc < NQ; qc++) {
          s[kt][qc] = (v4f){0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
      for (int x = 0; x < D / 32; x++)
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
          const v8bf k = kr[kt][x / (E / 8)].operand(x % (E / 8), attn_power_value(kp[kt]));
#pragma unroll
          for (int qc = 0; qc < NQ; qc++) s[kt][qc] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[qc][x], s[kt][qc], 0, 0, 0);
        }
      load(false, min(c + 1, c1 - 1), kr, kp);
      const bool edge = key0 + 32 > clear || (LOCAL && key0 < reach.every);
      // values into LDS, rows of bf16
      uint32_t odd = 0;
#pragma unroll
      for (int kt = 0; kt < 2; kt++) {
        uint8_t *row = values + (16 * kt + c16) * LD + 2 * E * g;
        const bool there = key0 + 16 * kt + c16 < r.kv;
#pragma unroll
        for (int x = 0; x < D / 32; x++) {
          v4i v = __builtin_bit_cast(v4i, vr[kt][x / (E / 8)].operand(x % (E / 8), attn_power_value(vp[kt])));
          if (edge) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t bad = no_numbers((uint32_t)v[i]);
              odd |= there ? bad : 0;
              v[i] = there ? v[i] & (int)~bad : 0;
            }
          }
          *(v4i *)(row + 8 * E * (x / (E / 8)) + 16 * (x % (E / 8))) = v;
        }
      }
      load(true, min(c + 1, c1 - 1), vr, vp);
      blocks(min(c + 2, c1 - 1));
      float scl = scale;
      if (__builtin_expect(edge, 0)) {
        attn_hide(a, r, sight, key0, scale, s);
        scl = 1.f;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      v8bf p[1][NQ], v[DT];
#pragma unroll
      for (int i = 0; i < 3; i++) v[i] = attn_values<LD>(read_at, i);
      st.template softmax<2>(s, scl, LOCAL ? edge || sure : edge || c == c0, p);
      sure = edge;
      attn_add_values<3, 1, LD>(st, read_at, p, v);
      if (__builtin_expect(edge && __any(odd != 0), 0)) attn_add_no_numbers<NQ, DT, C>(a, r, sight, table, kh, key0, 32, st);
      __builtin_amdgcn_wave_barrier();
    }
    // the wavefronts' results, each scaled to the common maximum, a quarter of the columns to each wavefront
    __syncthreads();
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) {
      const float l = over_groups(st.l[qc], true);
      if (g == 0) {
        sh_m[w][16 * qc + c16] = st.m[qc];
        sh_l[w][16 * qc + c16] = l;
      }
#pragma unroll
      for (int dt = 0; dt < DT; dt++) *(v4f *)(lds + (((size_t)w * DT + dt) * NQ + qc) * 1024 + lane * 16) = st.o[dt][qc];
    }
    __syncthreads();
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) {
      const int row = 16 * qc + c16;
      float m = sh_m[of_head][row], l = 0.f, f[SHARE];
#pragma unroll
      for (int i = 1; i < SHARE; i++) m = fmaxf(m, sh_m[of_head + HEADS * i][row]);
#pragma unroll
      for (int i = 0; i < SHARE; i++) {
        f[i] = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sh_m[of_head + HEADS * i][row] - m);
        l += sh_l[of_head + HEADS * i][row] * f[i];
      }
#pragma unroll
      for (int x = 0; x < DT / SHARE; x++) {
        const int dt = part_of_unit * (DT / SHARE) + x;
        v4f o = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < SHARE; i++) o += *(const v4f *)(lds + (((size_t)(of_head + HEADS * i) * DT + dt) * NQ + qc) * 1024 + lane * 16) * f[i];
        attn_store<ROWS, D>(a, r, kh, m_tile, row, 16 * dt + 4 * g, whole, part * HEADS + of_head, o, m, l);
      }
    }
    __syncthreads();
  });
}

// ---- staging in LDS (the two kernels below) ---------------------------------------------------------------------------
// Rows of a stage are 32 bytes longer than their values, so that reads of operands spread over the banks.  TPR
// threads write a row, 16 bytes of it at a time; which row thread group i takes is chosen so that the rows of one write fall into different
// banks as well: four rows 4 apart, or of bytes widened to 32 apart 0, 1, 8 and 9.  Of 4-bit codes, whose threads write a row's pieces further apart, rows
// are taken in order: a write's 16-byte pieces fall on every other group of banks, each twice.  Counted: no conflicts in the kernel of many rows on a bf16
// cache; in the one of 128 rows 2.7 of 10.1 million cycles at which LDS is read or written on an e4m3 cache, 2.7 of 10.0 in 4 bits; in the one of many rows 1.7
// of 9.7 in 4 bits.
template <int C, int TPR>
__device__ __forceinline__ int attn_stage_row(int i) {
  if (C == MOE_DTYPE_FP4) return i;
  if (C == MOE_DTYPE_FP8) return TPR == 4 ? (i & ~15) | (i & 1) | (i & 2) << 2 | (i >> 1 & 6) : i;
  return TPR == 4 ? (i & ~15) | (i & 3) << 2 | (i >> 2 & 3) : (i & ~15) | (i & 1) << 3 | (i >> 1 & 7);
}
template <int TPR, int NU, typename Piece>
__device__ __forceinline__ void attn_put(uint8_t *at, const Piece (&raw)[NU], uint32_t power) {
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int h = 0; h < Piece::E / 8; h++) *(v8bf *)(at + 2 * Piece::E * TPR * u + 16 * h) = raw[u].operand(h, attn_power_value(power));
}
// The same for values.  edge: the unit holds new tokens' values or ends the request, or has keys that only some rows see: what
// is no number becomes 0 and is told, what is beyond the end (there: this row is not) becomes 0.
template <int TPR, int NU, typename Piece>
__device__ __forceinline__ void attn_put_values(uint8_t *at, const Piece (&raw)[NU], uint32_t power, bool edge, bool there, int *any_odd) {
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int h = 0; h < Piece::E / 8; h++) {
      v4i v = __builtin_bit_cast(v4i, raw[u].operand(h, attn_power_value(power)));
      if (__builtin_expect(edge, 0)) {
        uint32_t odd = 0;
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const uint32_t bad = no_numbers((uint32_t)v[x]);
          odd |= there ? bad : 0;
          v[x] = there ? v[x] & (int)~bad : 0;
        }
        if (odd) *any_odd = 1;
      }
      *(v4i *)(at + 2 * Piece::E * TPR * u + 16 * h) = v;
    }
}

// ---- more rows: the wavefronts take the rows, and share the keys ---------------------------------------------------------
// Up to about 128 rows to a cached key both the bytes and the products count.  A workgroup stages 64 keys and values at a time in
// LDS, two stages of them, and every wavefront takes its rows past all of them, one barrier a stage; 16s of rows go to the wavefronts in turn, so that
// a tile that is not full keeps all at work (57 requests of about 145 rows: 108 us, 117 with neighbouring 16s together).  The bytes of the stage after
// that wait in registers (of two stages after it: no faster).  32 trees of up to 16 tokens over up to 8001 e4m3 keys: 69.5 us, 2.4 TB/s and
// 361 TFLOP/s; without the work on the stages 54, without the stages 56: two workgroups to a compute unit overlap the two in part, and
// LDS and registers hold no third.  (Codes are widened before they go to LDS, so an e4m3 cache has the stages of a bf16 one, and a 4-bit
// cache too: the same trees over half the bytes take 63 us and a join of 5 to 8, bound by the products, the widening and the stages.)
template <int D, int C, bool LOCAL, int NQ>
__global__ __launch_bounds__(256, 2) void attn_rows_kernel(const AttnArgs a) {
  constexpr int ROWS = 64 * NQ, UNIT = 64, DT = D / 16, LD = 2 * D + 32, STAGE = 2 * UNIT * LD;
  using Piece = AttnPiece<C, C == MOE_DTYPE_FP4 ? D / 8 : 16>;
  constexpr int BYTES = attn_row_bytes(C, D), TPR = 4, NU = BYTES / (Piece::BYTES * TPR);    // a row's threads; a thread's pieces of its row
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];
  __shared__ int any_odd;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c16 = lane & 15;
  attn_go<ROWS, UNIT, LOCAL, 1>(a, [&](const AttnRequest r, int b, int kh, int m_tile, int c0, int c1, bool whole, int part) {
    const int32_t *table = a.tables + (size_t)b * a.table_stride;
    const float factor = a.scale * (a.k_scale ? a.k_scale[kh] : 1.f) * 1.4426950408889634f, scale = fabsf(factor);
    const int clear = a.masks ? r.prefix : r.prefix + m_tile * ROWS / a.G + 1;      // keys below it are seen by every row
    const AttnReach reach = attn_reach<ROWS, UNIT, LOCAL>(a, r, m_tile);            // (and from reach.every on)
    const int last = c1 - 1;
    const int stage_row = attn_stage_row<C, TPR>(tid / TPR), piece = tid % TPR;
    uint8_t *const stage_at = lds + stage_row * LD + 2 * Piece::E * piece;
    Piece kr[NU], vr[NU];
    uint32_t kp = 0, vp = 0;                           // their powers of two
    int block;                                         // of the unit that is asked for next
    const auto key_of = [&](int unit) {
      const int c = min(unit, last), key = reach.unit(c) * UNIT + stage_row;
      return min(LOCAL ? reach.read(key) : key, r.kv - 1);
    };
    const auto is_edge = [&](int unit) { return (reach.unit(unit) + 1) * UNIT > clear || (LOCAL && reach.unit(unit) * UNIT < reach.every); };
    const auto ask = [&](int unit) {
      const int key = key_of(unit);
      const uint8_t *ka = attn_row<BYTES>(a, a.k_cache, a.k_block_bytes, block, kh, key) + Piece::BYTES * piece;
      const uint8_t *va = attn_row<BYTES>(a, a.v_cache, a.v_block_bytes, block, kh, key) + Piece::BYTES * piece;
#pragma unroll
      for (int u = 0; u < NU; u++) {
        kr[u].load(ka + Piece::BYTES * TPR * u);
        vr[u].load(va + Piece::BYTES * TPR * u);
      }
      if (C == MOE_DTYPE_FP4) {
        kp = attn_power<D>(a, a.k_powers, a.k_powers_block, block, kh, key, Piece::E * piece);
        vp = attn_power<D>(a, a.v_powers, a.v_powers_block, block, kh, key, Piece::E * piece);
      }
      block = attn_block(a, table, key_of(unit + 1));
    };
    const auto put = [&](int unit) {
      attn_put<TPR, NU>(stage_at + (unit & 1) * STAGE, kr, kp);
      attn_put_values<TPR, NU>(stage_at + (unit & 1) * STAGE + UNIT * LD, vr, vp, is_edge(unit), reach.unit(unit) * UNIT + stage_row < r.kv, &any_odd);
    };
    if (tid == 0) any_odd = 0;
    block = attn_block(a, table, key_of(c0));
    const auto begin = [&] {
      ask(c0);
      __syncthreads();
      put(c0);
      ask(c0 + 1);
      __syncthreads();
    };
    // the next stage's bytes from registers to LDS, the one's after those asked for
    const auto end_stage = [&](int c) {
      put(c + 1);
      ask(c + 2);
      __syncthreads();
    };
    const auto take = [&](auto sixteens) {
      constexpr int N = decltype(sixteens)::value, AHEAD = N == 2 && C == MOE_DTYPE_BF16 ? (LOCAL ? 1 : 2) : 3;     // (as the registers allow: 2 of LOCAL spills)
      v8bf q[N][D / 32];
      AttnSight<N, LOCAL> sight;
      attn_queries<N, D, 8, LOCAL, 64>(a, r, kh, m_tile * ROWS + 16 * w, factor, q, sight);
      AttnState<N, DT> st;
      st.clear();
      begin();
      bool sure = true;                                // the next keys may be the first that a row sees
      for (int c = c0; c < c1; c++) {
        const uint8_t *stage = lds + (c & 1) * STAGE;
        const bool edge = is_edge(c);
        v4f s[4][N];
        attn_scores<AHEAD, 4, LD>(stage + c16 * LD + 16 * g, q, s);
        const uint8_t *read_at = stage + UNIT * LD + (4 * g + c16 / 4) * LD + 8 * (c16 % 4);
        v8bf p[2][N], va[2 * DT];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) va[i] = attn_values<LD>(read_at, i);
        float scl = scale;
        if (__builtin_expect(edge, 0)) {
          attn_hide(a, r, sight, reach.unit(c) * UNIT, scale, s);
          scl = 1.f;
        }
        st.template softmax<4>(s, scl, LOCAL ? edge || sure : edge || c == c0, p);
        sure = edge;
        attn_add_values<AHEAD, 2, LD>(st, read_at, p, va);
        end_stage(c);
      }
      if (__builtin_expect(any_odd, 0)) {
        for (int c = LOCAL ? c0 : max(c0, clear / UNIT); c < c1; c++)      // the units whose values were looked at
          if (is_edge(c)) attn_add_no_numbers<N, DT, C>(a, r, sight, table, kh, reach.unit(c) * UNIT, UNIT, st);
      }
#pragma unroll
      for (int qc = 0; qc < N; qc++) {
        const float l = over_groups(st.l[qc], true);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
          attn_store<ROWS, D>(a, r, kh, m_tile, 16 * w + 64 * qc + c16, 16 * dt + 4 * g, whole, part, st.o[dt][qc], st.m[qc], l);
      }
    };
    // the tile's 16s of rows go to the wavefronts in turn, so that a tile that is not full still keeps all of them at work
    const int rows = r.n * a.G - m_tile * ROWS - 16 * w;
    if (NQ == 2 && rows > 64) take(std::integral_constant<int, NQ>());
    else if (rows > 0) take(std::integral_constant<int, 1>());
    else {                                             // a wavefront without rows only helps with the bytes
      begin();
      for (int c = c0; c < c1; c++) end_stage(c);
    }
    __syncthreads();
  });
}

// ---- many rows: two groups of wavefronts, one at the products while the other is at the exponentials ---------------------
// The matrix cores and the vector unit of a SIMD work at the same time only for different wavefronts, and two that share every barrier
// would always want the same one.  So wavefronts 4 to 7, one on each SIMD beside one of 0 to 3, run the same steps a slot later:
//   slot      0          1          2                     3
//   first     scores 0   weigh 0    scores 1, values 0    weigh 1 ...
//   second    -          scores 0   weigh 0               scores 1, values 0 ...
// A barrier ends a slot.  While it weighs unit c a wavefront also stages its share of the keys of c + 1 and the values of c, the
// second group's a unit further on, so that each stage is whole a slot before the first group needs it and is written when the second
// group has left it (two stages of each).  The 16s of rows go to the wavefronts in turn here too.
// Two chunks of 1021 tokens over 8190 keys: 219 to 238 us, 843 to 913 TFLOP/s where a large product alone reaches 1254; without the reads of
// operands from LDS 5 % less, without the exponentials 5 to 8 %, without staging 10 to 17 %.  Counted for a SIMD: the matrix cores are busy 196
// thousand clocks, the vector unit 220 thousand, of about 460 thousand: the two still add up more than they overlap.
// 16 trees of up to 64 tokens over up to 12288 keys: 119 to 124 us, 600 to 622 TFLOP/s (tiles that are not full, and a join of 12 us).
// LOCAL: the chunks in a window of 1024 58 us, 520 TFLOP/s of what the rows see (tiles of 64 tokens over 17 units for 16 units' worth of keys, then
// the way to the first unit), 66 over e4m3 and 63 over 4 bits; the trees in a window of 4095 87 to 92 us over each cache, of which 75 and a join of 10.5
// over 4 bits (97 to 100 us and 700 to 730 TFLOP/s where all texts are equally long).
template <int D, int C, bool LOCAL, int NQ>
__global__ __launch_bounds__(512, 2) void attn_pairs_kernel(const AttnArgs a) {
  constexpr int ROWS = 128 * NQ, UNIT = 64, DT = D / 16, X = D / 32, LD = 2 * D + 32, HALF = UNIT * LD;
  using Piece = AttnPiece<C, C == MOE_DTYPE_FP4 ? 8 : 16>;
  constexpr int BYTES = attn_row_bytes(C, D), TPR = BYTES / Piece::BYTES < 8 ? BYTES / Piece::BYTES : 8, NU = BYTES / (Piece::BYTES * TPR);
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * HALF];
  __shared__ int any_odd;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c16 = lane & 15;
  const int late = __builtin_amdgcn_readfirstlane(w) >> 2;
  attn_go<ROWS, UNIT, LOCAL, 1>(a, [&](const AttnRequest r, int b, int kh, int m_tile, int c0, int c1, bool whole, int part) {
    const int32_t *table = a.tables + (size_t)b * a.table_stride;
    const float factor = a.scale * (a.k_scale ? a.k_scale[kh] : 1.f) * 1.4426950408889634f, scale = fabsf(factor);
    const int clear = a.masks ? r.prefix : r.prefix + m_tile * ROWS / a.G + 1;      // keys below it are seen by every row
    const AttnReach reach = attn_reach<ROWS, UNIT, LOCAL>(a, r, m_tile);            // (and from reach.every on)
    const int last = c1 - 1;
    const int i = tid / TPR, piece = tid % TPR, stage_row = attn_stage_row<C, TPR>(i);
    const bool stages = i < UNIT;                      // (narrow rows take fewer threads)
    uint8_t *const stage_at = lds + stage_row * LD + 2 * Piece::E * piece;
    Piece kr[NU], vr[NU];
    uint32_t kp = 0, vp = 0;                           // their powers of two
    int block, block_v;                                // of the key, of the value that is asked for next
    const auto key_of = [&](int unit) {
      const int c = min(unit, last), key = reach.unit(c) * UNIT + stage_row;
      return min(LOCAL ? reach.read(key) : key, r.kv - 1);
    };
    const auto is_edge = [&](int unit) { return (reach.unit(unit) + 1) * UNIT > clear || (LOCAL && reach.unit(unit) * UNIT < reach.every); };
    const auto ask = [&](bool values, int blk, int unit, Piece (&to)[NU], uint32_t &power) {
      const int key = key_of(unit);
      const uint8_t *at = attn_row<BYTES>(a, values ? a.v_cache : a.k_cache, values ? a.v_block_bytes : a.k_block_bytes, blk, kh, key) + Piece::BYTES * piece;
#pragma unroll
      for (int u = 0; u < NU; u++) to[u].load(at + Piece::BYTES * TPR * u);
      if (C == MOE_DTYPE_FP4)
        power = attn_power<D>(a, values ? a.v_powers : a.k_powers, values ? a.v_powers_block : a.k_powers_block, blk, kh, key, Piece::E * piece);
    };
    const auto put_keys = [&](int unit) {
      if (stages) attn_put<TPR, NU>(stage_at + (unit & 1) * HALF, kr, kp);
    };
    const auto put_values = [&](int unit) {
      if (stages)
        attn_put_values<TPR, NU>(stage_at + (2 + (unit & 1)) * HALF, vr, vp, is_edge(unit), reach.unit(unit) * UNIT + stage_row < r.kv, &any_odd);
    };
    // keys of unit c + 1 and values of c into LDS, the next of both asked for
    const auto stage = [&](int c) {
      put_keys(c + 1);
      put_values(c);
      ask(false, block, c + 2, kr, kp);
      ask(true, block_v, c + 1, vr, vp);
      block_v = block;
      block = attn_block(a, table, key_of(c + 3));
    };

    if (tid == 0) any_odd = 0;
    block = attn_block(a, table, key_of(c0));
    const auto begin = [&] {
      ask(false, block, c0, kr, kp);
      ask(true, block, c0, vr, vp);
      block = block_v = attn_block(a, table, key_of(c0 + 1));
      put_keys(c0);
      ask(false, block, c0 + 1, kr, kp);
      block = attn_block(a, table, key_of(c0 + 2));
      __syncthreads();
      if (late) {                                        // slot 0
        stage(c0);
        __syncthreads();
      }
    };
    const auto take = [&](auto sixteens) {
      constexpr int N = decltype(sixteens)::value;
      v8bf q[N][X];
      AttnSight<N, LOCAL> sight;
      attn_queries<N, D, 8, LOCAL, 128>(a, r, kh, m_tile * ROWS + 16 * w, factor, q, sight);
      AttnState<N, DT> st;
      st.clear();
      begin();
      v4f s[4][N];
      attn_scores<4, 4, LD>(lds + (c0 & 1) * HALF + c16 * LD + 16 * g, q, s);
      __syncthreads();
      bool sure = true;                                // the next keys may be the first that a row sees
      for (int c = c0; c < c1; c++) {
        stage(c + late);
        const bool edge = is_edge(c);
        float scl = scale;
        if (__builtin_expect(edge, 0)) {
          attn_hide(a, r, sight, reach.unit(c) * UNIT, scale, s);
          scl = 1.f;
        }
        v8bf p[2][N], v[2 * DT];
        st.template softmax<4>(s, scl, LOCAL ? edge || sure : edge || c == c0, p);
        sure = edge;
        __syncthreads();
        attn_scores<4, 4, LD>(lds + ((c + 1) & 1) * HALF + c16 * LD + 16 * g, q, s);       // (past the last unit: of no use)
        const uint8_t *at = lds + (2 + (c & 1)) * HALF + (4 * g + c16 / 4) * LD + 8 * (c16 % 4);
#pragma unroll
        for (int x = 0; x < 4; x++) v[x] = attn_values<LD>(at, x);
        attn_add_values<4, 2, LD>(st, at, p, v);
        __syncthreads();
      }
      if (!late) __syncthreads();
      if (__builtin_expect(any_odd, 0)) {
        for (int c = LOCAL ? c0 : max(c0, clear / UNIT); c < c1; c++)      // the units whose values were looked at
          if (is_edge(c)) attn_add_no_numbers<N, DT, C>(a, r, sight, table, kh, reach.unit(c) * UNIT, UNIT, st);
      }
#pragma unroll
      for (int qc = 0; qc < N; qc++) {
        const float l = over_groups(st.l[qc], true);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
          attn_store<ROWS, D>(a, r, kh, m_tile, 16 * w + 128 * qc + c16, 16 * dt + 4 * g, whole, part, st.o[dt][qc], st.m[qc], l);
      }
    };
    const int rows = r.n * a.G - m_tile * ROWS - 16 * w;           // the 16s of rows in turn, as above
    if (rows > 128) take(std::integral_constant<int, NQ>());
    else if (rows > 0) take(std::integral_constant<int, 1>());
    else {                                             // a wavefront without rows only helps with the bytes
      begin();
      __syncthreads();
      for (int c = c0; c < c1; c++) {
        stage(c + late);
        __syncthreads();
        __syncthreads();
      }
      if (!late) __syncthreads();
    }
    __syncthreads();
  });
}

// ---- which kernel -------------------------------------------------------------------------------------------------------
// By the rows to a cached key that a request has on average, and by whether there is work for large tiles at all.  Measured, in us, 4 cache
// heads of 128, bf16 (e4m3); B requests of n tokens, 8 query heads a cache head, L keys:
//   rows  B x n x L            16 rows    64           128          256
//   8     64 x 1 x 8192        135 (81)
//   24    64 x 3 x 8192        134 (73)   123 (70)     126 (78)                     (16: with two 16s of rows a wavefront)
//   48    64 x 6 x 8192                   127 (76)     130 (92)     126 (110)
//   96    32 x 12 x 8192                  141 (116)    139 (104)    133 (117)
//   192   16 x 24 x 8192                  164          106          95
//   512   16 x 64 x 8192                  221          176          162
//   512   4 x 64 x 2048                   38 (39)      55 (54)      54 (55)
//   512   1 x 64 x 8192                   42 (43)      85 (85)      54 (55)
//   512   16 x 64 x 512                   29           37           37
//   512   4 x 64 x 8192                   70 (73)      78 (79)      74 (75)
//   2048  4 x 256 x 512, causal           54           42           43
//   400   1 x 400 x 2048, causal, no shared heads
//                                         29           33           37
// Large tiles read a key for more rows, small ones are more stretches at work and fewer, smaller parts to join.  Up to so many products of
// row and key the latter counts.  16 rows: two workgroups to a compute unit
// for e4m3, whose loads are half as long (256 requests of 2048 keys: 90 us with 512 workgroups, 105 with 256; bf16 146 and 141).
// Lengths are on the device, so the rule takes the table's width for them, and the average over all B requests for a request's rows.  Where these
// mislead it the call is right, but slower, us:
//   4 x 64 x 2048 with a table of 8192: 42 (38 in tiles of 64 rows); 1 x 64 x 8192 with one of 131072: 54 (43)
//   4 x 64 x 2048 beside 252 idle requests: 72;  511 x 1 x 1000 and a prompt of 512 in one call: 1613 (206 and 42 in two), 255 x 1 x 2048 and one
//   of 1024: 530.  (16 rows for the prompt: as many passes over its keys, and the walk)
// The walk along the line takes its time too: a piece of a causal request adds up all tiles of the request (attn_head_units), so that a prompt of 8192
// tokens from its start takes 1610 us of which 760 are the walk's, and requests without tokens are passed one by one (two single tokens over
// 2048 keys: 17, with 4000 idle requests between them 54).
// 4 bits: keys are cheaper to read than to unpack, so that tiles of 128 pay from 33 rows on (32 requests over 8001 keys, 64 and 128 rows a tile: 59 and 59 us
// at 32 rows, 66 and 64 at 48, 76 and 69 at 64).
// LOCAL kernels of more rows go by the same table, with the window's keys where those are fewer (16 x 64 tokens in a window of 1024, 64, 128 and 256
// rows: 46, 49 and 52 us; 32 x 64: 84, 63 and 61).  Those of 16 rows read two neighbouring heads' keys together, wider pieces of memory with fewer parts to join, where keys
// are many, and one head's where two would leave workgroups without a tile; and they have 512 workgroups where these find a tile each.  Us, 8
// cache heads, one and two heads with 256 workgroups, one and two with 512:
//   B x keys              bf16, 128               e4m3, 128               e4m3, 64                4 bits, 128             4 bits, 64
//   256 x up to 8192                                                      419  373  462  269                              498  411  462  297
//   64 x up to 8192       253  242  263  252      168  158  164  144      126  107  114   84      154  137  139  113      119  107  113   77
//   16 x up to 8192       82   73   84   76       51   48   48   46       32   29   35   27       41   40   40   37       34   32   31   29
//   128 x up to 1024      96   94   89   90       79   66   61   55       52   42   41   34       70   58   53   48       55   45   42   37
//   32 x up to 2048       47   45   49   49       34   32   29   30       26   25   23   22       34   32   29   30       27   25   24   24
//   256 x 1028 (window)                                                   124  104  102  72                               125  105  102  69
//   128 x 1028            122  114  114  113      89   74   72   69       64   53   55   38       80   71   64   51       66   53   42   37
//   64 x 1028             74   69   73   76       46   39   40   41       35   27   23   26       42   36   32   35       32   29   25   28
//   16 x 1028             23   26   28   29       19   21   21   21       15   16   16   17       19   21   21   22       16   16   17   19
//   1 x 32767, 4 heads    34   37   38   49       20   23   20   23       18   19   18   19       20   24   20   23       18   20   18   20
struct AttnPlan {
  int rows, groups;                    // rows of a tile; workgroups, a multiple of 8
  float cut;
  int heads;                           // cache heads of a workgroup (of 16 rows)
};
inline AttnPlan attn_plan(int T, int Hq, int Hkv, int B, int cache_dtype, bool local, bool trees, int64_t keys) {
  const int64_t rows = B > 0 ? ((int64_t)T * (Hq / Hkv) + B - 1) / B : 1;
  if (rows <= 16) {
    const bool bf16 = cache_dtype == MOE_DTYPE_BF16;
    if (!local) return {16, bf16 ? 256 : 512, 0.0625f, 1};
    const int64_t tiles = (int64_t)B * Hkv, all = tiles * keys;
    const int heads = Hkv % 2 == 0 && tiles >= 64 && all >= (bf16 ? 3 << 17 : 3 << 18) ? 2 : 1;
    const bool more = bf16 ? tiles / heads >= 512 : tiles < 64 || tiles > 128 || all > 1 << 18;
    return {16, more ? 512 : 256, 0.0625f, heads};
  }
  if (rows <= (cache_dtype == MOE_DTYPE_FP4 ? 32 : 64) || (int64_t)T * Hq <= (trees ? 20000000 : 8000000) / (keys > 0 ? keys : 1)) return {64, 512, 0.125f, 1};
  if (rows <= 128) return {128, 512, 0.125f, 1};
  return {256, 256, 0.25f, 1};
}
// what a plan's launches leave for each other: the stretches' parts, their maxima and sums, the records
inline size_t attn_workspace(const AttnPlan &p, int D) {
  const size_t rows = (size_t)p.rows * p.heads, parts = 2 * p.groups;
  return align_up(parts * rows * D * 4, 256) + align_up(parts * rows * 8, 256) + p.groups * 32;
}
// the keys that a row sees at most, where there is room for so many
inline int64_t attn_seen(int64_t room, int window, int sinks) {
  const int64_t most = window ? (int64_t)window + sinks : room;
  return most < room ? most : room;
}

constexpr int attn_cache_bits(int cache_dtype) { return cache_dtype == MOE_DTYPE_BF16 ? 16 : cache_dtype == MOE_DTYPE_FP8 ? 8 : 4; }

// What both entry points check and hand to their kernels.  scales: fp32 of each cache head, or a 4-bit cache's powers of two, whose blocks lie
// *_scale_stride bytes apart.  window 0: none; local: for the LOCAL kernels.  A call with nothing to do: MOE_OK and plan.rows 0.
inline int attn_arguments(const void *q_bf16, int64_t q_stride, int T, int Hq, int Hkv, int D, const void *k_cache, const void *v_cache, int cache_dtype,
                          int n_blocks, int64_t k_block_stride, int64_t v_block_stride, int page_size, const int32_t *block_tables,
                          int64_t table_stride, int table_width, const int32_t *kv_lens, const int32_t *cu_tokens, int B, const int64_t *masks,
                          float scale, const void *k_scale, const void *v_scale, int64_t k_scale_stride, int64_t v_scale_stride, int window,
                          int sinks, bool local, void *out_bf16, float *lse, void *workspace, size_t workspace_bytes, AttnPlan &plan, AttnArgs &a) {
  plan.rows = 0;
  const bool four = cache_dtype == MOE_DTYPE_FP4;
  if (T < 0 || B < 0 || B > MOE_MAX_REQUESTS || Hq < 1 || Hkv < 1 || Hq > 4096 || Hq % Hkv || (D != 64 && D != 128) || window < 0 || sinks < 0) return MOE_E_SHAPE;
  const int64_t row = (int64_t)Hkv * D;
  if (n_blocks < 0 || page_size < 1 || page_size > MOE_MAX_PAGE || (page_size & (page_size - 1)) || k_block_stride < page_size * row ||
      v_block_stride < page_size * row || table_width < 0 || (B > 1 && table_stride < table_width) || q_stride < (int64_t)Hq * D ||
      (int64_t)table_width * page_size >= (1ll << 31) || (int64_t)T * Hq >= (1ll << 31))
    return MOE_E_SHAPE;
  if (k_block_stride >= (1ll << 31) || v_block_stride >= (1ll << 31) || row >= (1 << 22)) return MOE_E_SHAPE;
  if (four && (k_scale_stride < page_size * row / 32 || v_scale_stride < page_size * row / 32 || k_scale_stride >= (1ll << 31) || v_scale_stride >= (1ll << 31)))
    return MOE_E_SHAPE;
  if (q_stride % 8 || k_block_stride % (four ? 32 : 16) || v_block_stride % (four ? 32 : 16)) return MOE_E_ALIGN;
  if (T == 0) return MOE_OK;
  if (!q_bf16 || !out_bf16 || !cu_tokens || !workspace || (B && !kv_lens)) return MOE_E_NULL;
  if (B && table_width && n_blocks && (!block_tables || !k_cache || !v_cache || (four && (!k_scale || !v_scale)))) return MOE_E_NULL;
  for (const void *p : {q_bf16, k_cache, v_cache, (const void *)out_bf16})
    if ((uintptr_t)p % 16) return MOE_E_ALIGN;
  if ((uintptr_t)workspace % 256) return MOE_E_ALIGN;
  const int64_t room = (int64_t)table_width * page_size, seen = attn_seen(room, window, sinks);
  AttnPlan p = attn_plan(T, Hq, Hkv, B, cache_dtype, local, masks != nullptr, seen);
  // (A workspace that moe_tree_attention would take is enough here too: then one head to a workgroup.)
  if (workspace_bytes < attn_workspace(p, D)) p = attn_plan(T, Hq, Hkv, B, cache_dtype, false, masks != nullptr, seen);
  if (workspace_bytes < attn_workspace(p, D)) return MOE_E_WORKSPACE;
  const int64_t most_units = ((int64_t)T * (Hq / Hkv) / p.rows + B) * Hkv * ((room + 63) / 64);
  if (most_units >= (1ll << 31)) return MOE_E_SHAPE;
  const size_t parts = 2 * p.groups;
  const int bits = attn_cache_bits(cache_dtype);
  uint8_t *const ws = (uint8_t *)workspace;
  a = AttnArgs{(const uint16_t *)q_bf16, q_stride, T, Hq, Hkv, Hq / Hkv, B, n_blocks, __builtin_ctz(page_size), n_blocks ? table_width : 0,
               (const uint8_t *)k_cache, (const uint8_t *)v_cache, (uint32_t)(k_block_stride * bits / 8), (uint32_t)(v_block_stride * bits / 8), table_stride,
               block_tables, kv_lens, cu_tokens, masks, scale, four ? nullptr : (const float *)k_scale, four ? nullptr : (const float *)v_scale,
               (uint16_t *)out_bf16, lse, p.groups, p.cut, (float *)workspace, (float *)(ws + align_up(parts * p.rows * p.heads * D * 4, 256)),
               (int32_t *)(ws + align_up(parts * p.rows * p.heads * D * 4, 256) + align_up(parts * p.rows * p.heads * 8, 256)), (uint32_t)most_units,
               window ? window : 0x7fffffff, sinks, four ? (const uint8_t *)k_scale : nullptr, four ? (const uint8_t *)v_scale : nullptr,
               (uint32_t)k_scale_stride, (uint32_t)v_scale_stride};
  plan = p;
  return MOE_OK;
}

// The main launch of a plan's kernel.  (The join, which knows nothing of the cache, is launched by attn_join.)
template <int D, int C, bool LOCAL>
void attn_main(const AttnArgs &a, const AttnPlan &plan, hipStream_t st) {
  if (plan.rows == 16 && plan.heads == 1) attn_keys_kernel<D, C, LOCAL, 1, 1><<<a.groups, 256, 0, st>>>(a);
  else if (plan.rows == 16) {
    if constexpr (LOCAL) attn_keys_kernel<D, C, LOCAL, 1, 2><<<a.groups, 256, 0, st>>>(a);
  }
  else if (plan.rows == 64) attn_rows_kernel<D, C, LOCAL, 1><<<a.groups, 256, 0, st>>>(a);
  else if (plan.rows == 128) attn_rows_kernel<D, C, LOCAL, 2><<<a.groups, 256, 0, st>>>(a);
  else attn_pairs_kernel<D, C, LOCAL, 2><<<a.groups, 512, 0, st>>>(a);
}
void attn_join(const AttnArgs &a, const AttnPlan &plan, int D, hipStream_t st);

}  // namespace moe
