// What a request asks of its logits before a token is drawn:
//
//   n    how often the request has generated a token, its history and the row's own drafted path;  heard: so or in its prompt
//   x    -> heard ? (x > 0 ? x / repetition : x repetition) : x
//        -> x - frequency n - presence [n > 0]
//        -> x + bias of the token                          (of a token named twice the last)
//        -> -inf unless the grammar allows the token
//
// fp32, one rounding at the end.  Bound by bytes: logits once in, once out.  A workgroup takes a segment of a row.  It
// counts the history's tokens that lie in the segment in LDS, so that no counter per vocabulary entry exists in memory, and a bit per token
// says which were touched.  A row streams through registers, is stored as it is (but for what its grammar forbids) without waiting for the
// counts, and the threads that stored the few touched values then store those once more.
// 64 rows of 131072 fp32 values with up to 8192 tokens of history: 22 to 23 us, 13 without the histories (3.0 and 5.3 TB/s); 1275 rows of 100003
// bf16 values, 128 requests' trees, every other row with a grammar: 143 us, 94 with neither (3.6 and 5.4 TB/s).  What histories cost is the
// comparisons of every token in every segment and the counting, about 25 instructions a token.  (LDS atomics of all lanes instead of a branch, and a list of
// the touched tokens in place of the bits, took 5 to 15 % longer.  Up to four rows of a request to a workgroup, which then counts once for
// them: 156 us for the 143, and 25 for 10 where there are 155 rows of 32000 values.)
// Histories of one token only, or filled up with -1, cost up to 1.7 times as much in segments of 64 KB, where lanes wait for each other at one counter:
// equal tokens are added up first only where 4 tokens of every thread, 4096 there, lie behind the prompt as a whole (38 us for the 22; bf16 22 for 13;
// segments of 24 KB 73 for 83).
#include <math.h>
#include <type_traits>
#include "moe_common.h"
#include "rows_clash.h"
#include "../../include/moe_hip.h"

namespace moe {

struct LogitArgs {
  const void *in;
  void *out;
  int64_t in_stride, out_stride;
  int T, V, B, L, bf16, segments;
  const int32_t *cu, *history;
  int64_t history_stride;
  const int32_t *history_lens, *prompt_lens;
  const int64_t *tokens, *masks;
  const float *repetition, *frequency, *presence;
  const int32_t *bias_ids;
  int64_t bias_ids_stride;
  const float *bias;
  int64_t bias_stride;
  int n_bias;
  const int32_t *allowed;
  int64_t allowed_stride;
  int allowed_rows;
  const int32_t *allowed_row;
};

// a counter: bit 0 heard in the prompt, bits 1 .. 20 how often generated, above them 1 + the place of the last bias that names the token
constexpr uint32_t kOnce = 2, kHeard = 1, kBiasShift = 21, kCounts = (1u << kBiasShift) - 1;

template <int SEG>
struct LogitTable {
  uint32_t count[SEG + 8];             // of token first - 8 + i: a group of 16 bytes may begin up to 7 tokens before the segment.  (Those of
                                       // ids below 0 and beyond the vocabulary are never read.)
  uint32_t touched[SEG / 32 + 2];
  __device__ __forceinline__ void touch(uint32_t place) { atomicOr(&touched[place >> 5], 1u << (place & 31)); }
  __device__ __forceinline__ void add(int64_t place, uint32_t what) {
    if (place < 0 || place >= SEG + 8) return;
    atomicAdd(&count[place], what);
    touch(place);
  }
};

typedef uint16_t __attribute__((aligned(1))) any_u16;

// BYTES of a row to a workgroup: BYTES / 16 groups of 16 bytes, P of them to a thread.
template <int BYTES, int THREADS, bool BF16>
__global__ __launch_bounds__(THREADS) void adjust_logits_kernel(const LogitArgs a) {
  constexpr int N = BF16 ? 8 : 4, E = BF16 ? 2 : 4, SEG = BYTES / E;             // values of 16 bytes; bytes of one
  constexpr int P = BYTES / (16 * THREADS), ALL = (1 << N) - 1;
  struct Group {
    uint32_t w[4], let;                // let: the grammar's bits for its values
  };
  __shared__ __attribute__((aligned(16))) LogitTable<SEG> s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int seg = blockIdx.x % a.segments;
  const int first = seg * SEG, from = first - 8;       // the segment's first token, for a row that begins on 16 bytes; the first counter's
  const int t = (int)(blockIdx.x / a.segments);

  // A row's groups begin on 16 bytes of memory: where the row does not, the first one begins `before` values earlier.  Of most segments all
  // groups lie within the row (inside); of the others some have values before or behind it, which are taken value by value.
  const uint8_t *in = (const uint8_t *)a.in + t * a.in_stride * E;
  uint8_t *out = (uint8_t *)a.out + t * a.out_stride * E;
  const int before = (int)((uintptr_t)in % 16) / E;
  const bool inside = first >= before && first - before + SEG <= a.V;
  const auto token_of = [&](int p) { return first + (p * THREADS + tid) * N - before; };
  const int grammar = !a.allowed ? -1 : a.allowed_row ? a.allowed_row[t] : t;
  const uint32_t *words = grammar >= 0 && grammar < a.allowed_rows ? (const uint32_t *)a.allowed + grammar * a.allowed_stride : nullptr;
  const int last_bits = (a.V + 31) / 32 * 4 - 2;       // a row of the grammar's last two bytes
  const auto bits_at = [&](int v) {
    const int at = min(v >> 3, last_bits);
    return (uint32_t)*(const any_u16 *)((const uint8_t *)words + at) >> (v - 8 * at) & ALL;
  };
  const auto store = [&](uint8_t *out, int v, bool same, const uint32_t (&w)[4]) {
    if (same) {
      *(v4i *)(out + (uint32_t)v * (uint32_t)E) = (v4i){(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    } else {
#pragma unroll
      for (int k = 0; k < N; k++) {
        if (BF16) ((uint16_t *)out)[(uint32_t)(v + k)] = (uint16_t)(w[k / 2] >> (16 * (k & 1)));
        else ((uint32_t *)out)[(uint32_t)(v + k)] = w[k];
      }
    }
  };

  Group now[P];
#pragma unroll
  for (int p = 0; p < P; p++) {
    const int v = token_of(p);
    now[p].let = ALL;
    if (inside || (v >= 0 && v + N <= a.V)) {
      const v4i raw = *(const v4i *)(in + (uint32_t)v * (uint32_t)E);
#pragma unroll
      for (int i = 0; i < 4; i++) now[p].w[i] = (uint32_t)raw[i];
    }
  }
  if (words) {
#pragma unroll
    for (int p = 0; p < P; p++) {
      const int v = token_of(p);
      if (inside || (v >= 0 && v + N <= a.V)) now[p].let = bits_at(v);
    }
  }

  // The row's request: the last one that begins at t or before.
  int b = t, begin = t, end = t + 1;
  if (a.cu) {
    int lo = 0, hi = a.B;                              // 64 places at a time
    while (lo < hi) {
      const int step = (hi - lo + 63) / 64, at = lo + (1 + lane) * step;
      const int past = __popcll(__ballot(at <= hi && a.cu[min(at, hi)] <= t));
      hi = min(lo + (past + 1) * step - 1, hi);
      lo += past * step;
    }
    b = lo < a.B && a.cu[lo] <= t ? lo : a.B;
    begin = b < a.B ? max(a.cu[b], 0) : t;
    end = b < a.B ? min(a.cu[b + 1], a.T) : t;
  }
  const bool none = b >= a.B;                          // a row of no request passes as it is
  // The history's first tokens are asked for together with its length and the penalties: one trip to memory.
  const int32_t *ids = a.history + (none ? 0 : b * a.history_stride);
  const bool heard = !none && a.history && a.L > 0;
  // (Four neighbours to a lane: histories are read by every segment, and single values took more loads than the logits.)
  v4i asked_for = {-1, -1, -1, -1};
  const bool whole = (uintptr_t)ids % 16 == 0;
  const auto ask = [&](int i0) {
    const int i = i0 + 4 * tid;
    if (whole && i + 4 <= a.L) {
      asked_for = *(const v4i *)(ids + i);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) asked_for[j] = i + j < a.L ? ids[i + j] : -1;
    }
  };
  if (heard) ask(0);
  const float rep = !none && a.repetition ? a.repetition[b] : 1.f, freq = !none && a.frequency ? a.frequency[b] : 0.f,
              pres = !none && a.presence ? a.presence[b] : 0.f;
  const int len = heard && a.history_lens ? min(a.history_lens[b], a.L) : a.L, asked = heard && a.prompt_lens ? min(a.prompt_lens[b], len) : 0;
  // the drafted tokens on the row's path: those that its mask names, 64 at the most, or those up to its own
  const uint64_t mask = !none && a.masks ? (uint64_t)a.masks[t] : 0;
  const bool drafted = !none && a.tokens && a.masks && tid < 64 && begin + tid < end && (mask >> tid & 1);
  const int64_t draft = drafted ? a.tokens[begin + tid] : 0;
  for (int i = tid; i < SEG / 4 + 2; i += THREADS) *(v4i *)&s.count[4 * i] = (v4i){0, 0, 0, 0};
  for (int i = tid; i < SEG / 32 + 2; i += THREADS) s.touched[i] = 0;

  // The row as it is, but for what its grammar forbids: this waits for nothing but the row.
  const bool same = (uintptr_t)out % 16 == (uintptr_t)in % 16, moved = a.out != a.in;
  if (none) words = nullptr;
#pragma unroll
  for (int p = 0; p < P; p++) {
    const int v = token_of(p);
    uint32_t (&w)[4] = now[p].w;
    if (inside || (v >= 0 && v + N <= a.V)) {
      if (words) {
        const uint32_t let = now[p].let;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (BF16) {
            const uint32_t keep = ((uint32_t)((int)(let << (31 - 2 * i)) >> 31) & 0xffffu) | ((uint32_t)((int)(let << (30 - 2 * i)) >> 31) & 0xffff0000u);
            w[i] = (w[i] & keep) | (0xff80ff80u & ~keep);
          } else {
            w[i] = let >> i & 1 ? w[i] : 0xff800000u;
          }
        }
      } else {
        now[p].let = ALL;
      }
      if (moved || words) store(out, v, same, w);
    } else {
      for (int k = max(v, 0); k < min(v + N, a.V); k++) {
        const bool may = !words || words[k >> 5] >> (k & 31) & 1;
        if (BF16) ((uint16_t *)out)[k] = may ? ((const uint16_t *)in)[k] : 0xff80;
        else ((uint32_t *)out)[k] = may ? ((const uint32_t *)in)[k] : 0xff800000u;
      }
    }
  }

  const float less = 1.0f / rep;
  const bool counts = rep != 1.f || freq != 0.f || pres != 0.f;
  if (none || !(counts || a.n_bias)) return;
  __syncthreads();
  if (a.n_bias) {
    for (int i = tid; i < a.n_bias; i += THREADS) {
      const uint32_t place = (uint32_t)(a.bias_ids[b * a.bias_ids_stride + i] - from);
      if (place >= SEG + 8) continue;
      atomicMax(&s.count[place], (uint32_t)(i + 1) << kBiasShift);
      s.touch(place);
    }
    __syncthreads();
  }
  if (heard && counts) {
    for (int i = 0; i < len; i += 4 * THREADS) {
      const v4i id = asked_for;
      if (i + 4 * THREADS < len) ask(i + 4 * THREADS);                 // (on their way while these are counted)
      const bool said = i >= asked && i + 4 * THREADS <= len, prompt = i + 4 * THREADS <= asked;       // (elsewhere threads differ)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t place = (uint32_t)(id[j] - from);
        if (place >= SEG + 8) continue;
        const int at = i + 4 * tid + j;
        const uint64_t here = __ballot(true);
        if ((said || prompt) && __popcll(here) > 40) {     // a text that repeats itself: so many additions at one address take as many turns
          const uint64_t like = __ballot(place == (uint32_t)__builtin_amdgcn_readfirstlane(place));
          if (like >> lane & 1) {
            if (lane == __builtin_ctzll(like)) {
              if (prompt) atomicOr(&s.count[place], kHeard);
              else atomicAdd(&s.count[place], (uint32_t)__popcll(like) * kOnce);
              s.touch(place);
            }
            continue;
          }
        }
        if (said || (at >= asked && at < len)) atomicAdd(&s.count[place], kOnce);
        else if (at < asked) atomicOr(&s.count[place], kHeard);
        s.touch(place);
      }
    }
  }
  if (counts && a.tokens) {
    if (drafted) s.add(draft - from, kOnce);
    if (!a.masks)
      for (int i = begin + tid; i <= t; i += THREADS) s.add(a.tokens[i] - from, kOnce);
  }
  __syncthreads();

  // The touched values, each by the thread that has just stored it.
  const auto adjusted = [&](float x, uint32_t c) {
    if (c & kCounts) {
      const float n = (float)((c & kCounts) >> 1);
      x = x * (x > 0.f ? less : rep) - (n > 0.f ? fmaf(freq, n, pres) : 0.f);
    }
    if (c >> kBiasShift) x += a.bias[b * a.bias_stride + (c >> kBiasShift) - 1];
    return x;
  };
  uint32_t hit[P];
#pragma unroll
  for (int p = 0; p < P; p++) {
    const int at = (p * THREADS + tid) * N - before + 8;             // the first one's counter
    const uint32_t lo = s.touched[at >> 5], hi = s.touched[(at >> 5) + 1];
    hit[p] = __builtin_amdgcn_alignbit(hi, lo, at & 31) & ALL;
  }
#pragma unroll
  for (int p = 0; p < P; p++) {
    const int v = token_of(p), at = (p * THREADS + tid) * N - before + 8;
    if (inside || (v >= 0 && v + N <= a.V)) {
      const v4i w = {(int)now[p].w[0], (int)now[p].w[1], (int)now[p].w[2], (int)now[p].w[3]};
      uint32_t left = hit[p] & now[p].let;
      while (left) {                                   // (few, if any: a wavefront passes as often as one of its lanes has hits)
        const int k = __builtin_ctz(left);
        left &= left - 1;
        const int word = BF16 ? k >> 1 : k;
        const uint32_t low = word & 1 ? w[1] : w[0], high = word & 1 ? w[3] : w[2], one = word & 2 ? high : low;
        const float x = adjusted(BF16 ? __uint_as_float(one >> (16 * (k & 1)) << 16) : __uint_as_float(one), s.count[at + k]);
        if (BF16) ((uint16_t *)out)[(uint32_t)(v + k)] = (uint16_t)pack2_bf16(x, 0.f);
        else ((float *)out)[(uint32_t)(v + k)] = x;
      }
    } else if (hit[p]) {
      for (int k = max(-v, 0); k < N && v + k < a.V; k++) {
        if (!s.count[at + k] || (words && !(words[(v + k) >> 5] >> ((v + k) & 31) & 1))) continue;
        const float x = adjusted(BF16 ? bf16_to_f32(((const uint16_t *)in)[v + k]) : ((const float *)in)[v + k], s.count[at + k]);
        if (BF16) ((uint16_t *)out)[v + k] = (uint16_t)pack2_bf16(x, 0.f);
        else ((float *)out)[v + k] = x;
      }
    }
  }
}

// Bytes of a row to a workgroup.  Large segments read the histories and zero the counters less often, small ones put more workgroups to work: of 24 KB
// three share a compute unit.  64 KB pay for long histories where they fill the chip once: a row's segments, times the rows, are workgroups of 1024
// threads, of which a bf16 one has a compute unit's LDS for itself; a few more than 256 take a second turn.  Two whole turns still pay where
// histories are longer.  Us, with the workgroups of 64 KB:
//                                                               16 KB     24        64
//   1 row of 131072 bf16, 4096 tokens of history      4         6.5       7.1       8.0
//   32 of 131072 bf16, 8192                           128       11.1      11.4      11.7
//   36 of 131072 bf16, 8192                           144       13.9      11.7      11.8
//   40 of 131072 bf16, 8192                           160       13.9      12.1      11.5
//   64 of 131072 bf16, 8192                           256       18.6      15.8      13.2
//   256 of 32000 bf16, 8192                           256       21.1      17.6      14.5
//   32 of 131072 fp32, 8192                           256       16.6      14.5      12.1
//   64 of 131072 bf16, 2048                           256       12.7      12.0      12.2
//   66 of 131072 bf16, 4096                           264       16.3      14.3      18.6
//   72 of 131072 bf16, 8192                           288       20.8      18.6      21.7
//   96 of 131072 bf16, 8192                           384       24.2      21.3      22.7
//   160 of 100003 bf16, 4096                          640       25.7      23.9      35.0
//   56 of 131072 fp32, 8192                           448       24.0      21.1      20.8
//   500 of 32000 bf16, 8192                           500       33.3      29.4      27.0
//   64 of 131072 fp32, 8192                           512       26.3      22.8      21.1 to 22.8
//   64 of 131072 fp32, 4096                           512       21.6      19.5      20.0
//   128 of 131072 bf16, 8192                          512       29.4      25.6      24.1 to 25.3
//   128 of 131072 bf16, 4096                          512       25.0      22.1      22.2
//   66 of 131072 fp32, 8192                           528       27.5      23.7      27.3
//   514 of 5493 bf16 (205 trees), 300 biases                    14.2      14.9      32.6
//   155 of 32000 bf16 (16 trees), 2000                155       10.1      9.6       11.8
//   320 of 131072 fp32 (64 trees), 2000               2560      99        78        113
//   512 of 100003 bf16, 4096                          2048      73        64        98
//   1275 of 100003 bf16 (128 trees), 2048             5100      160       143       252
// wide: a row's values with room for those before its first 16 bytes; L: of the histories, 0 without any.
static int logit_segment(int64_t wide, int e, int T, int V, int L) {
  const int64_t work = (int64_t)T * V * e, large = (wide * e + 65535) / 65536 * T;
  if (L >= 4096 && large >= 160 && large <= 256 && work >= (10 << 20)) return 65536;
  if (L >= 8192 && large >= 448 && large <= 512 && work >= (27 << 20)) return 65536;
  return work < (6 << 20) ? 16384 : 24576;
}

}  // namespace moe

extern "C" int moe_adjust_logits(void *stream, const void *logits, int dtype, int64_t row_stride, int T, int V, const int32_t *cu_tokens, int B,
                                 const int32_t *history, int64_t history_stride, int L, const int32_t *history_lens, const int32_t *prompt_lens,
                                 const int64_t *tokens, const int64_t *masks, const float *repetition, const float *frequency,
                                 const float *presence, const int32_t *bias_ids, int64_t bias_ids_stride, const float *bias, int64_t bias_stride,
                                 int n_bias, const int32_t *allowed, int64_t allowed_stride, int n_allowed, const int32_t *allowed_rows,
                                 void *out, int64_t out_stride) {
  using namespace moe;
  if (dtype != MOE_DTYPE_F32 && dtype != MOE_DTYPE_BF16) return MOE_E_MODE;
  if (T < 0 || V < 1 || V >= (1 << 30) || B < 0 || L < 0 || n_bias < 0 || n_bias > MOE_MAX_BIASES || row_stride < V || out_stride < V || n_allowed < 0 ||
      (!cu_tokens && B != T) || (int64_t)L + T >= (1 << 20))
    return MOE_E_SHAPE;
  if ((history && history_stride < L) || (n_bias && (bias_ids_stride < n_bias || bias_stride < n_bias)) ||
      (allowed && (allowed_stride < (V + 31) / 32 || (!allowed_rows && n_allowed != T))))
    return MOE_E_SHAPE;
  if (T == 0) return MOE_OK;
  if (!logits || !out || (n_bias && (!bias_ids || !bias)) || (masks && !tokens)) return MOE_E_NULL;
  const int64_t e = dtype == MOE_DTYPE_BF16 ? 2 : 4;
  if ((uintptr_t)logits % e || (uintptr_t)out % e) return MOE_E_ALIGN;
  const auto over = [&](const void *p, int64_t rows, int64_t stride, int64_t row, int size) {      // out lies over an input of such rows
    return rows_clash(out, out_stride * e, V * e, T, p, stride * size, row * size, rows);
  };
  if ((!(logits == out && (row_stride == out_stride || T == 1)) && over(logits, T, row_stride, V, (int)e)) || over(cu_tokens, 1, 0, B + 1ll, 4) ||
      over(history, B, history_stride, L, 4) || over(tokens, 1, 0, T, 8) || over(masks, 1, 0, T, 8) || over(n_bias ? bias_ids : nullptr, B, bias_ids_stride, n_bias, 4) ||
      over(n_bias ? bias : nullptr, B, bias_stride, n_bias, 4) || over(allowed, n_allowed, allowed_stride, (V + 31) / 32, 4) ||
      over(allowed ? allowed_rows : nullptr, 1, 0, T, 4))
    return MOE_E_MODE;
  for (const void *p : {(const void *)history_lens, (const void *)prompt_lens, (const void *)repetition, (const void *)frequency, (const void *)presence})
    if (over(p, 1, 0, B, 4)) return MOE_E_MODE;
  LogitArgs a{logits, out, row_stride, out_stride, T, V, B, L, dtype == MOE_DTYPE_BF16, 0, cu_tokens,
              history, history_stride, history_lens, prompt_lens, tokens, masks, repetition, frequency, presence, bias_ids, bias_ids_stride, bias,
              bias_stride, n_bias, allowed, allowed_stride, n_allowed, allowed_rows};
  hipStream_t st = (hipStream_t)stream;
  // (rows that begin on 16 bytes need no room for the values before)
  const int64_t wide = (uintptr_t)logits % 16 == 0 && (T == 1 || row_stride * e % 16 == 0) ? V : (int64_t)V + 16 / e - 1;
  const auto run = [&](auto bytes, auto threads) {
    constexpr int BYTES = decltype(bytes)::value, TH = decltype(threads)::value;
    a.segments = (int)((wide * e + BYTES - 1) / BYTES);
    const int64_t blocks = (int64_t)a.segments * T;
    if (blocks * TH >> 32) return MOE_E_SHAPE;         // (a launch has fewer than 2^32 threads)
    if (a.bf16) adjust_logits_kernel<BYTES, TH, true><<<(unsigned)blocks, TH, 0, st>>>(a);
    else adjust_logits_kernel<BYTES, TH, false><<<(unsigned)blocks, TH, 0, st>>>(a);
    return (int)hipGetLastError();
  };
  using std::integral_constant;
  const int bytes = logit_segment(wide, (int)e, T, V, history ? L : 0);
  if (bytes == 16384) return run(integral_constant<int, 16384>(), integral_constant<int, 512>());
  if (bytes == 65536) return run(integral_constant<int, 65536>(), integral_constant<int, 1024>());
  return run(integral_constant<int, 24576>(), integral_constant<int, 512>());
}

extern "C" int moe_adjust_logits_segment_bytes(int dtype, int T, int V, int L) {
  if ((dtype != MOE_DTYPE_F32 && dtype != MOE_DTYPE_BF16) || T < 1 || V < 1 || V >= (1 << 30) || L < 0) return 0;
  return moe::logit_segment(V, dtype == MOE_DTYPE_BF16 ? 2 : 4, T, V, L);
}
