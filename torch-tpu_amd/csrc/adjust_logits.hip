// What a request asks of its logits before a token is drawn:
//
//   n    how often the request has generated a token, its history and the row's own drafted path;  heard: so or in its prompt
//   x    -> heard ? (x > 0 ? x / repetition : x repetition) : x
//        -> x - frequency n - presence [n > 0]
//        -> x + bias of the token                          (of a token named twice the last)
//        -> -inf unless the grammar allows the token
//
// fp32, one rounding at the end.  Bound by bytes: logits once in, once out.  A workgroup takes a segment of the vocabulary for some rows.  It
// counts the history's tokens that lie in the segment in LDS, so that no counter per vocabulary entry exists in memory and histories, which are short
// beside the vocabulary, are read again by each segment.  Most tokens are touched by nothing: a bit of each says so, and their values pass
// as they are.
#include "moe_common.h"
#include "../../include/moe_hip.h"

namespace moe {

struct LogitArgs {
  const void *in;
  void *out;
  int64_t in_stride, out_stride;
  int T, V, B, L, bf16, rows, segments;        // rows: of a workgroup
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
  uint32_t count[SEG + 8];             // of token first - 8 + i: a group of 16 bytes may begin up to 7 tokens before the segment
  uint32_t touched[SEG / 32 + 2];
};

template <int SEG>
__device__ __forceinline__ void note(LogitTable<SEG> &s, int64_t place, uint32_t what) {
  if (place < 0 || place >= SEG + 8) return;
  atomicAdd(&s.count[place], what);
  atomicOr(&s.touched[place >> 5], 1u << (place & 31));
}

template <int SEG, bool BF16>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const LogitArgs a) {
  constexpr int N = BF16 ? 8 : 4, E = BF16 ? 2 : 4;    // values of 16 bytes; bytes of one
  __shared__ LogitTable<SEG> s;
  const int tid = threadIdx.x;
  const int seg = blockIdx.x % a.segments;
  const int64_t first = (int64_t)seg * SEG;            // the segment's first token, for a row that begins on 16 bytes
  const int t0 = (int)(blockIdx.x / a.segments) * a.rows, t1 = min(t0 + a.rows, a.T);
  int b = -1, begin = 0, end = 0;                      // the request whose history is counted, its rows
  uint64_t path = 0;                                   // the tokens of the tree that are counted
  for (int t = t0; t < t1; t++) {
    bool fresh = false;
    if (a.cu) {
      if (b < 0 || t >= end) {                         // the last request that begins at t or before
        int lo = 0, hi = a.B;
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if (a.cu[mid] <= t) lo = mid;
          else hi = mid - 1;
        }
        fresh = true;
        b = lo < a.B && a.cu[lo] <= t ? lo : a.B;
        begin = b < a.B ? max(a.cu[b], 0) : t;
        end = b < a.B ? min(a.cu[b + 1], a.T) : lo < a.B ? min(a.cu[lo], a.T) : a.T;
      }
    } else {
      fresh = true;
      b = t, begin = t, end = t + 1;
    }
    const bool none = b >= a.B;                        // a row of no request passes as it is
    const float rep = !none && a.repetition ? a.repetition[b] : 1.f, freq = !none && a.frequency ? a.frequency[b] : 0.f,
                pres = !none && a.presence ? a.presence[b] : 0.f;
    const bool counts = rep != 1.f || freq != 0.f || pres != 0.f;
    if (fresh) {
      __syncthreads();
      for (int i = tid; i < SEG + 8; i += 256) s.count[i] = 0;
      for (int i = tid; i < SEG / 32 + 2; i += 256) s.touched[i] = 0;
      __syncthreads();
      if (!none && a.n_bias) {
        for (int i = tid; i < a.n_bias; i += 256) {
          const int64_t place = (int64_t)a.bias_ids[b * a.bias_ids_stride + i] - first + 8;
          if (place < 0 || place >= SEG + 8) continue;
          atomicMax(&s.count[place], (uint32_t)(i + 1) << kBiasShift);
          atomicOr(&s.touched[place >> 5], 1u << (place & 31));
        }
        __syncthreads();
      }
      if (!none && counts && a.history) {
        const int len = min(max(a.history_lens ? a.history_lens[b] : a.L, 0), a.L), asked = a.prompt_lens ? a.prompt_lens[b] : 0;
        for (int i = tid; i < len; i += 256) {
          const int64_t place = (int64_t)a.history[b * a.history_stride + i] - first + 8;
          if (place < 0 || place >= SEG + 8) continue;
          if (i < asked) atomicOr(&s.count[place], kHeard);
          else atomicAdd(&s.count[place], kOnce);
          atomicOr(&s.touched[place >> 5], 1u << (place & 31));
        }
      }
      path = 0;
      if (!none && counts && a.tokens && !a.masks)     // what stands before the row
        for (int i = begin + tid; i < t; i += 256) note<SEG>(s, a.tokens[i] - first + 8, kOnce);
    }
    if (!none && counts && a.tokens) {
      if (a.masks) {
        const uint64_t mask = (uint64_t)a.masks[t];
        if (tid < 64 && begin + tid < end) {
          const int was = path >> tid & 1, is = mask >> tid & 1;
          if (was != is) note<SEG>(s, a.tokens[begin + tid] - first + 8, is ? kOnce : 0u - kOnce);
        }
        path = mask;
      } else if (tid == 0) {
        note<SEG>(s, a.tokens[t] - first + 8, kOnce);
      }
    }
    __syncthreads();
    // Groups of 16 bytes of memory: a row that does not begin on one has its first group `before` values earlier.
    const uint8_t *in = (const uint8_t *)a.in + t * a.in_stride * E;
    uint8_t *out = (uint8_t *)a.out + t * a.out_stride * E;
    const int before = (int)((uintptr_t)in % 16) / E;
    const bool same = (uintptr_t)out % 16 == (uintptr_t)in % 16;
    const int grammar = a.allowed && !none ? (a.allowed_row ? a.allowed_row[t] : t) : -1;
    const uint32_t *words = grammar >= 0 && grammar < a.allowed_rows ? (const uint32_t *)a.allowed + grammar * a.allowed_stride : nullptr;
    const int last_word = (a.V - 1) / 32;
    for (int i = tid; i < SEG / N; i += 256) {
      const int64_t v0 = first + (int64_t)i * N - before;
      if (v0 >= a.V) break;
      const int from = v0 < 0 ? (int)-v0 : 0, upto = v0 + N > a.V ? (int)(a.V - v0) : N;     // the group's values that are the row's
      if (from >= upto) continue;
      const bool full = from == 0 && upto == N;
      uint32_t raw[N];
      if (full) {
        const v4i w = *(const v4i *)(in + v0 * E);
#pragma unroll
        for (int k = 0; k < N; k++) raw[k] = BF16 ? (uint32_t)w[k / 2] >> (16 * (k & 1)) & 0xffff : (uint32_t)w[k];
      } else {
#pragma unroll
        for (int k = 0; k < N; k++) raw[k] = k >= from && k < upto ? (BF16 ? (uint32_t)((const uint16_t *)in)[v0 + k] : ((const uint32_t *)in)[v0 + k]) : 0;
      }
      const int at = i * N - before + 8;               // the first one's counter
      const uint32_t hit = (uint32_t)(((uint64_t)s.touched[(at >> 5) + 1] << 32 | s.touched[at >> 5]) >> (at & 31)) & ((1u << N) - 1);
      uint32_t let = (1u << N) - 1;
      if (words) {
        const int64_t w0 = v0 + from;
        const int w = (int)(w0 >> 5);
        let = (uint32_t)(((uint64_t)words[min(w + 1, last_word)] << 32 | words[w]) >> (w0 & 31)) << from & ((1u << N) - 1);
      }
      if (hit) {
#pragma unroll
        for (int k = 0; k < N; k++) {
          if (!(hit >> k & 1)) continue;
          const uint32_t c = s.count[at + k];
          float x = BF16 ? bf16_to_f32((uint16_t)raw[k]) : __uint_as_float(raw[k]);
          if (c & kCounts) {
            x = x > 0.f ? x / rep : x * rep;
            const float n = (float)((c & kCounts) >> 1);
            x = x - freq * n - (n > 0.f ? pres : 0.f);
          }
          if (c >> kBiasShift) x += a.bias[b * a.bias_stride + (c >> kBiasShift) - 1];
          raw[k] = BF16 ? f32_to_bf16(x) : __float_as_uint(x);
        }
      }
#pragma unroll
      for (int k = 0; k < N; k++)
        if (!(let >> k & 1)) raw[k] = BF16 ? 0xff80u : 0xff800000u;
      if (full && same) {
        v4i w;
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = BF16 ? (int)(raw[N / 4 * k] | raw[N / 4 * k + 1] << 16) : (int)raw[k];
        *(v4i *)(out + v0 * E) = w;
      } else {
#pragma unroll
        for (int k = 0; k < N; k++) {
          if (k < from || k >= upto) continue;
          if (BF16) ((uint16_t *)out)[v0 + k] = (uint16_t)raw[k];
          else ((uint32_t *)out)[v0 + k] = raw[k];
        }
      }
    }
    __syncthreads();
  }
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
  if (T < 0 || V < 1 || B < 0 || L < 0 || n_bias < 0 || n_bias > MOE_MAX_BIASES || row_stride < V || out_stride < V || n_allowed < 0 ||
      (!cu_tokens && B != T) || (int64_t)L + T >= (1 << 20))
    return MOE_E_SHAPE;
  if ((history && history_stride < L) || (n_bias && (bias_ids_stride < n_bias || bias_stride < n_bias)) ||
      (allowed && (allowed_stride < (V + 31) / 32 || (!allowed_rows && n_allowed != T))))
    return MOE_E_SHAPE;
  if (T == 0) return MOE_OK;
  if (!logits || !out || (n_bias && (!bias_ids || !bias)) || (masks && !tokens)) return MOE_E_NULL;
  const int64_t e = dtype == MOE_DTYPE_BF16 ? 2 : 4;
  if ((uintptr_t)logits % e || (uintptr_t)out % e) return MOE_E_ALIGN;
  const uint8_t *i0 = (const uint8_t *)logits, *o0 = (const uint8_t *)out;
  if (!(i0 == o0 && (row_stride == out_stride || T == 1)) && i0 < o0 + ((T - 1) * out_stride + V) * e && o0 < i0 + ((T - 1) * row_stride + V) * e)
    return MOE_E_MODE;
  constexpr int SEG = 8192;
  const int rows = B > 0 ? (T + B - 1) / B : 1;
  LogitArgs a{logits, out, row_stride, out_stride, T, V, B, L, dtype == MOE_DTYPE_BF16, rows < 16 ? rows : 16, (V + 7 + SEG - 1) / SEG, cu_tokens,
              history, history_stride, history_lens, prompt_lens, tokens, masks, repetition, frequency, presence, bias_ids, bias_ids_stride, bias,
              bias_stride, n_bias, allowed, allowed_stride, n_allowed, allowed_rows};
  const int64_t blocks = (int64_t)a.segments * ((T + a.rows - 1) / a.rows);
  if (blocks > 0x7fffffff) return MOE_E_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  if (a.bf16) adjust_logits_kernel<SEG, true><<<(unsigned)blocks, 256, 0, st>>>(a);
  else adjust_logits_kernel<SEG, false><<<(unsigned)blocks, 256, 0, st>>>(a);
  return (int)hipGetLastError();
}
