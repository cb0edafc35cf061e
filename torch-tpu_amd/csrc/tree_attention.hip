// Attention of new tokens over a paged cache: one token of each request, a tree of drafted ones, or a causal chunk.
//
//   token j of request b sees the cached keys [0, p), p = kv_len - n, and of the n new ones, which the cache holds as
//   well, those that its mask names (no masks: 0 .. j);   o = sum_key softmax(scale q.key) value
//
// One pass over the keys with the running maximum and sum of the softmax, both fp32, as is the output until its one
// rounding.  A token that sees nothing gives 0 and -inf.
#include <math.h>
#include <type_traits>
#include "moe_common.h"
#include "moe_layout.h"
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
// rows of tile m see keys below this
template <int ROWS>
__device__ __forceinline__ int attn_tile_end(const AttnArgs &a, const AttnRequest &r, int m) {
  if (a.masks || r.n == 1) return r.kv;
  return r.prefix + min(r.n, (min((m + 1) * ROWS, r.n * a.G) - 1) / a.G + 1);
}
template <int ROWS, int UNIT>
__device__ __forceinline__ int attn_head_units(const AttnArgs &a, const AttnRequest &r) {
  if (r.n <= 0 || r.prefix < 0) return 0;
  const int tiles = (r.n * a.G + ROWS - 1) / ROWS;
  if (a.masks || r.n == 1) return tiles * ((r.kv + UNIT - 1) / UNIT);
  int sum = 0;
  for (int m = 0; m < tiles; m++) sum += (attn_tile_end<ROWS>(a, r, m) + UNIT - 1) / UNIT;
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
        u = (attn_tile_end<ROWS>(a, r, m) + UNIT - 1) / UNIT;
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
template <int NQ>
struct AttnSight {
  uint64_t mask[NQ];                   // without masks: the last key seen
  // bit k: query qc sees key first_key + k
  __device__ __forceinline__ uint64_t from(const AttnArgs &a, const AttnRequest &r, int qc, int first_key) const {
    const auto first = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
    if (!a.masks) return first((int)mask[qc] + 1 - first_key);
    const int i = first_key - r.prefix;                // the first key's bit
    return first(r.kv - first_key) & (i >= 64 ? 0ull : i >= 0 ? mask[qc] >> i : i > -64 ? mask[qc] << -i | first(-i) : ~0ull);
  }
};

// Hides what a lane's queries do not see; the scores left are scaled already.
template <int NQ, int KT>
__device__ __forceinline__ void attn_hide(const AttnArgs &a, const AttnRequest &r, const AttnSight<NQ> &sight, int first_key, float c,
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

// 16 bytes of the cache -> operands of 8 bf16: themselves, or two of e4m3 codes
__device__ __forceinline__ v8bf attn_widen(const v4i raw, int half) {
  const uint32_t w0 = (uint32_t)raw[2 * half], w1 = (uint32_t)raw[2 * half + 1];
  const v4i w = {__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true))};
  return __builtin_bit_cast(v8bf, w);
}
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

// A value that is NaN or infinite would, times a probability of 0, reach rows that do not see its key.  Where new tokens are among
// the keys such values are staged as 0, and this adds them to the rows that do see them.
template <int NQ, int DT, bool FP8>
__device__ __forceinline__ void attn_add_no_numbers(const AttnArgs &a, const AttnRequest &r, const AttnSight<NQ> &sight, const int32_t *table,
                                                 int kh, int first_key, int keys, AttnState<NQ, DT> &st) {
  const int g4 = 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll 1
  for (int key = first_key; key < min(first_key + keys, r.kv); key++) {
    const uint8_t *row = attn_row<DT * (FP8 ? 16 : 32)>(a, a.v_cache, a.v_block_bytes, attn_block(a, table, key), kh, key);
    bool sees[NQ];
#pragma unroll
    for (int qc = 0; qc < NQ; qc++) sees[qc] = sight.from(a, r, qc, key) & 1;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int d = 16 * dt + g4 + i;
        float v = FP8 ? __builtin_amdgcn_cvt_f32_fp8((uint32_t)row[d], 0) : bf16_to_f32(((const uint16_t *)row)[d]);
        v = __builtin_isfinite(v) ? 0.f : v;
#pragma unroll
        for (int qc = 0; qc < NQ; qc++) st.o[dt][qc][i] += sees[qc] ? v : 0.f;
      }
  }
}

// a lane's queries as the scores' second operand: element j of step s is d = 32 s + 8 g + j, or with e4m3 keys, of which a lane reads
// 16 at a time, d = 64 (s / 2) + 16 g + 8 (s % 2) + j.  Its 16s of rows lie STEP apart.  Of the scores' factor the queries take the
// sign, so that the largest score is the largest product.
template <int NQ, int D, bool FP8, int STEP = 16>
__device__ __forceinline__ void attn_queries(const AttnArgs &a, const AttnRequest &r, int kh, int first_row, float factor, v8bf (&q)[NQ][D / 32],
                                             AttnSight<NQ> &sight) {
  const int lane = threadIdx.x & 63, g = lane >> 4, flip = factor < 0.f ? (int)0x80008000 : 0;
#pragma unroll
  for (int qc = 0; qc < NQ; qc++) {
    const int row = min(first_row + STEP * qc + (lane & 15), r.n * a.G - 1), j = row / a.G, h = kh * a.G + row - j * a.G;
    const uint16_t *src = a.q + (size_t)(r.t0 + j) * a.q_stride + (size_t)h * D;
#pragma unroll
    for (int s = 0; s < D / 32; s++) {
      const v4i w = *(const v4i *)(src + (FP8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g));
      q[qc][s] = __builtin_bit_cast(v8bf, w ^ flip);
    }
    sight.mask[qc] = a.masks ? (uint64_t)a.masks[r.t0 + j] : (uint64_t)(r.prefix + j);
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
template <int D, bool FP8, int NQ>
__global__ __launch_bounds__(256, 2) void attn_keys_kernel(const AttnArgs a) {
  constexpr int ROWS = 16 * NQ, UNIT = 128, DT = D / 16, LD = 2 * D + 32, P = FP8 ? D / 64 : D / 32;   // P: 16-byte pieces of a lane's key
  constexpr int kValues = 4 * 32 * LD, kMerge = 4 * DT * NQ * 64 * 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kValues > kMerge ? kValues : kMerge];
  __shared__ float sh_m[4][ROWS], sh_l[4][ROWS];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
  uint8_t *values = lds + w * 32 * LD;
  const uint8_t *read_at = values + (4 * g + c16 / 4) * LD + 8 * (c16 % 4);
  attn_walk<ROWS, UNIT>(a, [&](const AttnRequest r, int b, int kh, int m_tile, int c0, int c1, bool whole, int part) {
    const int32_t *table = a.tables + (size_t)b * a.table_stride;
    const float factor = a.scale * (a.k_scale ? a.k_scale[kh] : 1.f) * 1.4426950408889634f, scale = fabsf(factor);
    v8bf q[NQ][D / 32];
    AttnSight<NQ> sight;
    attn_queries<NQ, D, FP8>(a, r, kh, m_tile * ROWS, factor, q, sight);
    const int clear = a.masks ? r.prefix : r.prefix + m_tile * ROWS / a.G + 1;      // keys below it are seen by every row
    AttnState<NQ, DT> st;
    st.clear();
    // The block of a key is read two units ahead of the key, so that no load waits for another one.
    v4i kr[2][P], vr[2][P];
    int block[2];
    const auto key_of = [&](int unit, int kt) { return min(unit * UNIT + 32 * w + 16 * kt + c16, r.kv - 1); };
    const auto blocks = [&](int unit) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++) block[kt] = attn_block(a, table, key_of(unit, kt));
    };
    const auto load = [&](const uint8_t *cache, uint32_t block_bytes, int unit, v4i (&to)[2][P]) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++) {
        const uint8_t *row = attn_row<FP8 ? D : 2 * D>(a, cache, block_bytes, block[kt], kh, key_of(unit, kt)) + 16 * g;
#pragma unroll
        for (int p = 0; p < P; p++) to[kt][p] = *(const v4i *)(row + 64 * p);
      }
    };
    blocks(c0);
    load(a.k_cache, a.k_block_bytes, c0, kr);
    load(a.v_cache, a.v_block_bytes, c0, vr);
    blocks(min(c0 + 1, c1 - 1));
    for (int c = c0; c < c1; c++) {
      const int key0 = c * UNIT + 32 * w;
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
          const v8bf k = FP8 ? attn_widen(kr[kt][x / 2], x % 2) : __builtin_bit_cast(v8bf, kr[kt][FP8 ? 0 : x]);
#pragma unroll
          for (int qc = 0; qc < NQ; qc++) s[kt][qc] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[qc][x], s[kt][qc], 0, 0, 0);
        }
      load(a.k_cache, a.k_block_bytes, min(c + 1, c1 - 1), kr);
      const bool edge = key0 + 32 > clear;
      // values into LDS, rows of bf16
      uint32_t odd = 0;
#pragma unroll
      for (int kt = 0; kt < 2; kt++) {
        uint8_t *row = values + (16 * kt + c16) * LD + (FP8 ? 32 : 16) * g;
        const bool there = key0 + 16 * kt + c16 < r.kv;
#pragma unroll
        for (int x = 0; x < D / 32; x++) {
          v4i v = FP8 ? __builtin_bit_cast(v4i, attn_widen(vr[kt][x / 2], x % 2)) : vr[kt][FP8 ? 0 : x];
          if (edge) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t bad = no_numbers((uint32_t)v[i]);
              odd |= there ? bad : 0;
              v[i] = there ? v[i] & (int)~bad : 0;
            }
          }
          *(v4i *)(row + (FP8 ? 128 * (x / 2) + 16 * (x % 2) : 64 * x)) = v;
        }
      }
      load(a.v_cache, a.v_block_bytes, min(c + 1, c1 - 1), vr);
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
      st.template softmax<2>(s, scl, edge || c == c0, p);
      attn_add_values<3, 1, LD>(st, read_at, p, v);
      if (__builtin_expect(edge && __any(odd != 0), 0)) attn_add_no_numbers<NQ, DT, FP8>(a, r, sight, table, kh, key0, 32, st);
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
      float m = sh_m[0][row], l = 0.f, f[4];
#pragma unroll
      for (int i = 1; i < 4; i++) m = fmaxf(m, sh_m[i][row]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        f[i] = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sh_m[i][row] - m);
        l += sh_l[i][row] * f[i];
      }
#pragma unroll
      for (int x = 0; x < DT / 4; x++) {
        const int dt = w * (DT / 4) + x;
        v4f o = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; i++) o += *(const v4f *)(lds + (((size_t)i * DT + dt) * NQ + qc) * 1024 + lane * 16) * f[i];
        attn_store<ROWS, D>(a, r, kh, m_tile, row, 16 * dt + 4 * g, whole, part, o, m, l);
      }
    }
    __syncthreads();
  });
}

// ---- staging in LDS (the two kernels below) ---------------------------------------------------------------------------
// Rows of a stage are 32 bytes longer than their values, so that reads of operands spread over the banks.  TPR
// threads write a row, 16 bytes of it at a time; which row thread group i takes is chosen so that the rows of one write fall into different
// banks as well: four rows 4 apart, or of bytes widened to 32 apart 0, 1, 8 and 9.  Counted: no conflicts in the kernel of many rows on
// a bf16 cache; in the one of 128 rows on an e4m3 cache 2.7 of 10.1 million cycles at which LDS is read or written.
template <bool FP8, int TPR>
__device__ __forceinline__ int attn_stage_row(int i) {
  if (FP8) return TPR == 4 ? (i & ~15) | (i & 1) | (i & 2) << 2 | (i >> 1 & 6) : i;
  return TPR == 4 ? (i & ~15) | (i & 3) << 2 | (i >> 2 & 3) : (i & ~15) | (i & 1) << 3 | (i >> 1 & 7);
}
template <bool FP8, int TPR, int NU>
__device__ __forceinline__ void attn_put(uint8_t *at, const v4i (&raw)[NU]) {
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int h = 0; h < (FP8 ? 2 : 1); h++)
      *(v4i *)(at + (FP8 ? 32 : 16) * TPR * u + 16 * h) = FP8 ? __builtin_bit_cast(v4i, attn_widen(raw[u], h)) : raw[u];
}
// The same for values.  edge: the unit holds new tokens' values or ends the request: what is no number becomes 0 and is told, what
// is beyond the end (there: this row is not) becomes 0.
template <bool FP8, int TPR, int NU>
__device__ __forceinline__ void attn_put_values(uint8_t *at, const v4i (&raw)[NU], bool edge, bool there, int *any_odd) {
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int h = 0; h < (FP8 ? 2 : 1); h++) {
      v4i v = FP8 ? __builtin_bit_cast(v4i, attn_widen(raw[u], h)) : raw[u];
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
      *(v4i *)(at + (FP8 ? 32 : 16) * TPR * u + 16 * h) = v;
    }
}

// ---- more rows: the wavefronts take the rows, and share the keys ---------------------------------------------------------
// Up to about 128 rows to a cached key both the bytes and the products count.  A workgroup stages 64 keys and values at a time in
// LDS, two stages of them, and every wavefront takes its rows past all of them, one barrier a stage; 16s of rows go to the wavefronts in turn, so that
// a tile that is not full keeps all at work (57 requests of about 145 rows: 108 us, 117 with neighbouring 16s together).  The bytes of the stage after
// that wait in registers (of two stages after it: no faster).  32 trees of up to 16 tokens over up to 8001 e4m3 keys: 69.5 us, 2.4 TB/s and
// 361 TFLOP/s; without the work on the stages 54, without the stages 56: two workgroups to a compute unit overlap the two in part, and
// LDS and registers hold no third.  (Codes are widened before they go to LDS, so an e4m3 cache has the stages of a bf16 one.)
template <int D, bool FP8, int NQ>
__global__ __launch_bounds__(256, 2) void attn_rows_kernel(const AttnArgs a) {
  constexpr int ROWS = 64 * NQ, UNIT = 64, DT = D / 16, LD = 2 * D + 32, STAGE = 2 * UNIT * LD;
  constexpr int BYTES = FP8 ? D : 2 * D, TPR = 4, NU = BYTES / (16 * TPR);           // a row's threads; a thread's 16-byte pieces of its row
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];
  __shared__ int any_odd;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c16 = lane & 15;
  attn_walk<ROWS, UNIT>(a, [&](const AttnRequest r, int b, int kh, int m_tile, int c0, int c1, bool whole, int part) {
    const int32_t *table = a.tables + (size_t)b * a.table_stride;
    const float factor = a.scale * (a.k_scale ? a.k_scale[kh] : 1.f) * 1.4426950408889634f, scale = fabsf(factor);
    const int clear = a.masks ? r.prefix : r.prefix + m_tile * ROWS / a.G + 1;      // keys below it are seen by every row
    const int last = c1 - 1;
    const int stage_row = attn_stage_row<FP8, TPR>(tid / TPR), piece = tid % TPR;
    uint8_t *const stage_at = lds + stage_row * LD + (FP8 ? 32 : 16) * piece;
    v4i kr[NU], vr[NU];
    int block;                                         // of the unit that is asked for next
    const auto key_of = [&](int unit) { return min(min(unit, last) * UNIT + stage_row, r.kv - 1); };
    const auto ask = [&](int unit) {
      const uint8_t *ka = attn_row<BYTES>(a, a.k_cache, a.k_block_bytes, block, kh, key_of(unit)) + 16 * piece;
      const uint8_t *va = attn_row<BYTES>(a, a.v_cache, a.v_block_bytes, block, kh, key_of(unit)) + 16 * piece;
#pragma unroll
      for (int u = 0; u < NU; u++) {
        kr[u] = *(const v4i *)(ka + 16 * TPR * u);
        vr[u] = *(const v4i *)(va + 16 * TPR * u);
      }
      block = attn_block(a, table, key_of(unit + 1));
    };
    const auto put = [&](int unit) {
      attn_put<FP8, TPR, NU>(stage_at + (unit & 1) * STAGE, kr);
      attn_put_values<FP8, TPR, NU>(stage_at + (unit & 1) * STAGE + UNIT * LD, vr, (unit + 1) * UNIT > clear,
                                    unit * UNIT + stage_row < r.kv, &any_odd);
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
      constexpr int N = decltype(sixteens)::value, AHEAD = N == 2 && !FP8 ? 2 : 3;     // (as the registers allow)
      v8bf q[N][D / 32];
      AttnSight<N> sight;
      attn_queries<N, D, false, 64>(a, r, kh, m_tile * ROWS + 16 * w, factor, q, sight);
      AttnState<N, DT> st;
      st.clear();
      begin();
      for (int c = c0; c < c1; c++) {
        const uint8_t *stage = lds + (c & 1) * STAGE;
        const bool edge = (c + 1) * UNIT > clear;
        v4f s[4][N];
        attn_scores<AHEAD, 4, LD>(stage + c16 * LD + 16 * g, q, s);
        const uint8_t *read_at = stage + UNIT * LD + (4 * g + c16 / 4) * LD + 8 * (c16 % 4);
        v8bf p[2][N], va[2 * DT];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) va[i] = attn_values<LD>(read_at, i);
        float scl = scale;
        if (__builtin_expect(edge, 0)) {
          attn_hide(a, r, sight, c * UNIT, scale, s);
          scl = 1.f;
        }
        st.template softmax<4>(s, scl, edge || c == c0, p);
        attn_add_values<AHEAD, 2, LD>(st, read_at, p, va);
        end_stage(c);
      }
      if (__builtin_expect(any_odd, 0)) {
        const int from = max(c0, clear / UNIT) * UNIT;          // the first unit whose values were looked at
        attn_add_no_numbers<N, DT, FP8>(a, r, sight, table, kh, from, c1 * UNIT - from, st);
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
template <int D, bool FP8, int NQ>
__global__ __launch_bounds__(512, 2) void attn_pairs_kernel(const AttnArgs a) {
  constexpr int ROWS = 128 * NQ, UNIT = 64, DT = D / 16, X = D / 32, LD = 2 * D + 32, HALF = UNIT * LD;
  constexpr int BYTES = FP8 ? D : 2 * D, TPR = BYTES / 16 < 8 ? BYTES / 16 : 8, NU = BYTES / (16 * TPR);
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * HALF];
  __shared__ int any_odd;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c16 = lane & 15;
  const int late = __builtin_amdgcn_readfirstlane(w) >> 2;
  attn_walk<ROWS, UNIT>(a, [&](const AttnRequest r, int b, int kh, int m_tile, int c0, int c1, bool whole, int part) {
    const int32_t *table = a.tables + (size_t)b * a.table_stride;
    const float factor = a.scale * (a.k_scale ? a.k_scale[kh] : 1.f) * 1.4426950408889634f, scale = fabsf(factor);
    const int clear = a.masks ? r.prefix : r.prefix + m_tile * ROWS / a.G + 1;      // keys below it are seen by every row
    const int last = c1 - 1;
    const int i = tid / TPR, piece = tid % TPR, stage_row = attn_stage_row<FP8, TPR>(i);
    const bool stages = i < UNIT;                      // (narrow rows take fewer threads)
    uint8_t *const stage_at = lds + stage_row * LD + (FP8 ? 32 : 16) * piece;
    v4i kr[NU], vr[NU];
    int block, block_v;                                // of the key, of the value that is asked for next
    const auto key_of = [&](int unit) { return min(min(unit, last) * UNIT + stage_row, r.kv - 1); };
    const auto ask = [&](const uint8_t *cache, uint32_t block_bytes, int blk, int unit, v4i (&to)[NU]) {
      const uint8_t *at = attn_row<BYTES>(a, cache, block_bytes, blk, kh, key_of(unit)) + 16 * piece;
#pragma unroll
      for (int u = 0; u < NU; u++) to[u] = *(const v4i *)(at + 16 * TPR * u);
    };
    const auto put_keys = [&](int unit) {
      if (stages) attn_put<FP8, TPR, NU>(stage_at + (unit & 1) * HALF, kr);
    };
    const auto put_values = [&](int unit) {
      if (stages)
        attn_put_values<FP8, TPR, NU>(stage_at + (2 + (unit & 1)) * HALF, vr, (unit + 1) * UNIT > clear, unit * UNIT + stage_row < r.kv, &any_odd);
    };
    // keys of unit c + 1 and values of c into LDS, the next of both asked for
    const auto stage = [&](int c) {
      put_keys(c + 1);
      put_values(c);
      ask(a.k_cache, a.k_block_bytes, block, c + 2, kr);
      ask(a.v_cache, a.v_block_bytes, block_v, c + 1, vr);
      block_v = block;
      block = attn_block(a, table, key_of(c + 3));
    };

    if (tid == 0) any_odd = 0;
    block = attn_block(a, table, key_of(c0));
    const auto begin = [&] {
      ask(a.k_cache, a.k_block_bytes, block, c0, kr);
      ask(a.v_cache, a.v_block_bytes, block, c0, vr);
      block = block_v = attn_block(a, table, key_of(c0 + 1));
      put_keys(c0);
      ask(a.k_cache, a.k_block_bytes, block, c0 + 1, kr);
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
      AttnSight<N> sight;
      attn_queries<N, D, false, 128>(a, r, kh, m_tile * ROWS + 16 * w, factor, q, sight);
      AttnState<N, DT> st;
      st.clear();
      begin();
      v4f s[4][N];
      attn_scores<4, 4, LD>(lds + (c0 & 1) * HALF + c16 * LD + 16 * g, q, s);
      __syncthreads();
      for (int c = c0; c < c1; c++) {
        stage(c + late);
        const bool edge = (c + 1) * UNIT > clear;
        float scl = scale;
        if (__builtin_expect(edge, 0)) {
          attn_hide(a, r, sight, c * UNIT, scale, s);
          scl = 1.f;
        }
        v8bf p[2][N], v[2 * DT];
        st.template softmax<4>(s, scl, edge || c == c0, p);
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
        const int from = max(c0, clear / UNIT) * UNIT;          // the first unit whose values were looked at
        attn_add_no_numbers<N, DT, FP8>(a, r, sight, table, kh, from, c1 * UNIT - from, st);
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

// ---- joining ------------------------------------------------------------------------------------------------------------
// Row blocks of the tile that began in stretch blockIdx.x and went on in later ones: the parts in the stretches' order.  A row is taken by
// SPLIT groups of D / 4 lanes, each a share of the parts, which meet in LDS.  Rows of no request and of refused ones become 0.
template <int ROWS, int D, int SPLIT>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
  constexpr int lanes = D / 4, per_block = 256 / (lanes * SPLIT);
  __shared__ v4f sh_o[256];
  __shared__ float sh_m[256 / lanes], sh_l[256 / lanes];
  const int tid = threadIdx.x, group = tid / lanes, d = 4 * (tid % lanes), split = group % SPLIT;
  if (blockIdx.y == gridDim.y - 1) {
    const auto nothing = [&](int t) {
      for (int i = tid; i < a.Hq * lanes; i += 256) *(v2i *)(a.out + ((size_t)t * a.Hq * lanes + i) * 4) = (v2i){0, 0};
      if (a.lse)
        for (int i = tid; i < a.Hq; i += 256) a.lse[(size_t)t * a.Hq + i] = -INFINITY;
    };
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      const AttnRequest r = attn_request(a, b);
      if (r.prefix < 0)
        for (int j = 0; j < r.n; j++) nothing(r.t0 + j);
    }
    const int first = min(max(a.cu[0], 0), a.T), end = min(max(a.cu[a.B], 0), a.T);
    for (int t = blockIdx.x; t < first; t += gridDim.x) nothing(t);
    for (int t = end + (int)blockIdx.x; t < a.T; t += gridDim.x) nothing(t);
    return;
  }
  const int *rec = a.records + 8 * blockIdx.x;
  const int w1 = rec[0], kh = rec[3], m_tile = rec[4], side = rec[5], w0 = blockIdx.x;
  const AttnRequest r{rec[1], rec[2], 0, 0};
  if (w1 <= w0) return;
  const int in_tile = blockIdx.y * per_block + group / SPLIT, row = m_tile * ROWS + in_tile;
  if (m_tile * ROWS + (int)blockIdx.y * per_block >= r.n * a.G) return;
  const auto part = [&](int w) { return (size_t)(2 * w + (w == w0 ? side : 0)) * ROWS + in_tile; };
  float m = -INFINITY, l = 0.f;
  v4f o = (v4f){0.f, 0.f, 0.f, 0.f};
  if (row < r.n * a.G) {
    for (int first = w0 + split; first <= w1; first += 4 * SPLIT) {      // four parts asked for at a time (eight: slower where there are four)
      float pm[4], pl[4];
      v4f po[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const size_t at = part(min(first + i * SPLIT, w1));
        pm[i] = a.part_ml[at * 2], pl[i] = a.part_ml[at * 2 + 1];
        po[i] = *(const v4f *)(a.part_o + at * D + d);
      }
      const float before = m;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (first + i * SPLIT > w1) pm[i] = -INFINITY, pl[i] = 0.f, po[i] = (v4f){0.f, 0.f, 0.f, 0.f};
        m = fmaxf(m, pm[i]);
      }
      const float top = m == -INFINITY ? 0.f : m;      // (nothing seen so far: weights of 0, not of -inf + inf)
      const float f = __builtin_amdgcn_exp2f(before - top);
      l *= f;
      o *= f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float w = __builtin_amdgcn_exp2f(pm[i] - top);
        l += pl[i] * w;
        o += po[i] * w;
      }
    }
  }
  if (SPLIT > 1) {
    sh_o[tid] = o;
    if (d == 0) sh_m[group] = m, sh_l[group] = l;
    __syncthreads();
    if (split) return;
    m = sh_m[group];
#pragma unroll
    for (int i = 1; i < SPLIT; i++) m = fmaxf(m, sh_m[group + i]);
    l = 0.f;
    o = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SPLIT; i++) {
      const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sh_m[group + i] - m);
      l += sh_l[group + i] * f;
      o += sh_o[tid + i * lanes] * f;
    }
  }
  attn_store<ROWS, D>(a, r, kh, m_tile, in_tile, d, true, 0, o, m, l);
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
struct AttnPlan {
  int rows, groups;                    // rows of a tile; workgroups, a multiple of 8
  float cut;
};
static AttnPlan attn_plan(int T, int Hq, int Hkv, int B, int cache_dtype, bool trees, int64_t keys) {
  const int64_t rows = B > 0 ? ((int64_t)T * (Hq / Hkv) + B - 1) / B : 1;
  if (rows <= 16) return {16, cache_dtype == MOE_DTYPE_FP8 ? 512 : 256, 0.0625f};
  if (rows <= 64 || (int64_t)T * Hq <= (trees ? 20000000 : 8000000) / (keys > 0 ? keys : 1)) return {64, 512, 0.125f};
  if (rows <= 128) return {128, 512, 0.125f};
  return {256, 256, 0.25f};
}

}  // namespace moe

extern "C" size_t moe_tree_attention_workspace_bytes(int T, int Hq, int Hkv, int D, int B, int cache_dtype) {
  using namespace moe;
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 1 || B < 0 || (cache_dtype != MOE_DTYPE_BF16 && cache_dtype != MOE_DTYPE_FP8)) return 0;
  const AttnPlan plan = attn_plan(T, Hq, Hkv, B, cache_dtype, false, 1ll << 31);      // (shorter caches need no more)
  const size_t rows = plan.rows, parts = 2 * plan.groups;
  return align_up(parts * rows * D * 4, 256) + align_up(parts * rows * 8, 256) + plan.groups * 32;
}

extern "C" int moe_tree_attention_tile_rows(int T, int Hq, int Hkv, int B, int cache_dtype, int trees, int table_width, int page_size) {
  using namespace moe;
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || B < 0 || B > MOE_MAX_REQUESTS || (cache_dtype != MOE_DTYPE_BF16 && cache_dtype != MOE_DTYPE_FP8) ||
      table_width < 0 || page_size < 1 || page_size > MOE_MAX_PAGE || (page_size & (page_size - 1)))
    return 0;
  return attn_plan(T, Hq, Hkv, B, cache_dtype, trees != 0, (int64_t)table_width * page_size).rows;
}

extern "C" int moe_tree_attention(void *stream, const void *q_bf16, int64_t q_stride, int T, int Hq, int Hkv, int D,
                                  const void *k_cache, const void *v_cache, int cache_dtype, int n_blocks, int64_t k_block_stride,
                                  int64_t v_block_stride, int page_size, const int32_t *block_tables, int64_t table_stride,
                                  int table_width, const int32_t *kv_lens, const int32_t *cu_tokens, int B, const int64_t *masks,
                                  float scale, const float *k_scale, const float *v_scale, void *out_bf16, float *lse,
                                  void *workspace, size_t workspace_bytes) {
  using namespace moe;
  if (cache_dtype != MOE_DTYPE_BF16 && cache_dtype != MOE_DTYPE_FP8) return MOE_E_MODE;
  if (T < 0 || B < 0 || B > MOE_MAX_REQUESTS || Hq < 1 || Hkv < 1 || Hq > 4096 || Hq % Hkv || (D != 64 && D != 128)) return MOE_E_SHAPE;
  const int64_t row = (int64_t)Hkv * D;
  if (n_blocks < 0 || page_size < 1 || page_size > MOE_MAX_PAGE || (page_size & (page_size - 1)) || k_block_stride < page_size * row ||
      v_block_stride < page_size * row || table_width < 0 || (B > 1 && table_stride < table_width) || q_stride < (int64_t)Hq * D ||
      (int64_t)table_width * page_size >= (1ll << 31) || (int64_t)T * Hq >= (1ll << 31))
    return MOE_E_SHAPE;
  if (k_block_stride >= (1ll << 31) || v_block_stride >= (1ll << 31) || row >= (1 << 22)) return MOE_E_SHAPE;
  if (q_stride % 8 || k_block_stride % 16 || v_block_stride % 16) return MOE_E_ALIGN;
  if (T == 0) return MOE_OK;
  if (!q_bf16 || !out_bf16 || !cu_tokens || !workspace || (B && !kv_lens)) return MOE_E_NULL;
  if (B && table_width && n_blocks && (!block_tables || !k_cache || !v_cache)) return MOE_E_NULL;
  for (const void *p : {q_bf16, k_cache, v_cache, (const void *)out_bf16})
    if ((uintptr_t)p % 16) return MOE_E_ALIGN;
  if ((uintptr_t)workspace % 256) return MOE_E_ALIGN;
  if (workspace_bytes < moe_tree_attention_workspace_bytes(T, Hq, Hkv, D, B, cache_dtype)) return MOE_E_WORKSPACE;
  const int fp8 = cache_dtype == MOE_DTYPE_FP8, wide = fp8 ? 1 : 2;
  const AttnPlan plan = attn_plan(T, Hq, Hkv, B, cache_dtype, masks != nullptr, (int64_t)table_width * page_size);
  const int64_t most_units = ((int64_t)T * (Hq / Hkv) / plan.rows + B) * Hkv * (((int64_t)table_width * page_size + 63) / 64);
  if (most_units >= (1ll << 31)) return MOE_E_SHAPE;
  const size_t parts = 2 * plan.groups;
  AttnArgs a{(const uint16_t *)q_bf16, q_stride, T, Hq, Hkv, Hq / Hkv, B, n_blocks, __builtin_ctz(page_size), n_blocks ? table_width : 0,
             (const uint8_t *)k_cache, (const uint8_t *)v_cache, (uint32_t)(k_block_stride * wide), (uint32_t)(v_block_stride * wide), table_stride,
             block_tables, kv_lens, cu_tokens, masks, scale, k_scale, v_scale, (uint16_t *)out_bf16, lse, plan.groups, plan.cut, (float *)workspace,
             (float *)((uint8_t *)workspace + align_up(parts * plan.rows * D * 4, 256)),
             (int32_t *)((uint8_t *)workspace + align_up(parts * plan.rows * D * 4, 256) + align_up(parts * plan.rows * 8, 256)), (uint32_t)most_units};
  hipStream_t st = (hipStream_t)stream;
  using std::integral_constant;
  const auto run = [&](auto dim, auto narrow) {
    constexpr int Dc = decltype(dim)::value;
    constexpr bool F = decltype(narrow)::value;
    const auto join = [&](auto rows, auto split) {
      constexpr int R = decltype(rows)::value, S = decltype(split)::value;
      attn_join_kernel<R, Dc, S><<<dim3(a.groups, R * Dc * S / 1024 + 1), 256, 0, st>>>(a);
    };
    if (plan.rows == 16) {
      attn_keys_kernel<Dc, F, 1><<<a.groups, 256, 0, st>>>(a);
      join(integral_constant<int, 16>(), integral_constant<int, 8>());
    } else if (plan.rows == 64) {
      attn_rows_kernel<Dc, F, 1><<<a.groups, 256, 0, st>>>(a);
      join(integral_constant<int, 64>(), integral_constant<int, 2>());
    } else if (plan.rows == 128) {
      attn_rows_kernel<Dc, F, 2><<<a.groups, 256, 0, st>>>(a);
      join(integral_constant<int, 128>(), integral_constant<int, 1>());
    } else {
      attn_pairs_kernel<Dc, F, 2><<<a.groups, 512, 0, st>>>(a);
      join(integral_constant<int, 256>(), integral_constant<int, 1>());
    }
  };
  if (D == 64 && fp8) run(integral_constant<int, 64>(), integral_constant<bool, true>());
  else if (D == 64) run(integral_constant<int, 64>(), integral_constant<bool, false>());
  else if (fp8) run(integral_constant<int, 128>(), integral_constant<bool, true>());
  else run(integral_constant<int, 128>(), integral_constant<bool, false>());
  return (int)hipGetLastError();
}
