// logits.cu -- what happens to logits before the next token is chosen.
//
// For every row m and token v, in this order, in f32:
//   repetition  v anywhere in the row's history:      x > 0 ? x / r : x * r
//   frequency   x -= f * (times v was generated)
//   presence    x -= a, once, if v was generated
//   bias        x += the row's biases for v (in list order)
//   grammar     x = -inf where the row's mask has a 0 (whatever x was)
// and optionally the index of the row's largest result (the lowest such index; NaN
// never; -1 when nothing is above -inf).  "Generated" is the part of the history
// from prompt_lens on.
//
// One pass over the logits.  A CTA takes a chunk of one row that its threads hold in
// registers: NV 16-byte loads each, issued before anything else.  While they travel it
// goes once through the history: a bit per token that occurs, a list of those tokens,
// and per token a count (bit 15 or 31 = in the prompt, the rest = times generated;
// integer atomics, so any order gives the same counts).  The listed tokens (and those
// with a bias) are then worked out side by side, one per thread, and most tokens,
// which carry no bit, go through as they came.  (Working the marked tokens out where
// they are streamed costs every warp the longest of its lanes' paths: 105 us instead
// of 66 at 256 x 131071 f16 with 2048 tokens of history.)  The largest value is
// joined over a row's CTAs by a 64-bit maximum of (ordered value, ~index) and a
// counter; the last CTA writes the token and clears both.  Bound: HBM, 2 e bytes per
// logit + 1/8 for the mask; small calls by their launch.
#include <cuda_bf16.h>

#include "q4_common.cuh"
#include "q4_logits.cuh"
#include "q4_status.cuh"

namespace aria_q4 {

constexpr int kLogitThreads = 256;

template <int DT>
struct LogitType;
template <>
struct LogitType<0> {
  using T = float;
  static __device__ float get(T v) { return v; }
  static __device__ T put(float v) { return v; }
};
template <>
struct LogitType<1> {
  using T = __half;
  static __device__ float get(T v) { return __half2float(v); }
  static __device__ T put(float v) { return __float2half_rn(v); }
};
template <>
struct LogitType<2> {
  using T = __nv_bfloat16;
  static __device__ float get(T v) { return __bfloat162float(v); }
  static __device__ T put(float v) { return __float2bfloat16_rn(v); }
};

// monotone in x; every finite value and the infinities are > 0
__device__ __forceinline__ uint32_t logit_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// 32 bits of a bit array from bit i on (a word past the last is read: it exists)
__device__ __forceinline__ uint32_t bits_from(const uint32_t* w, int i) {
  return __funnelshift_r(w[i >> 5], w[(i >> 5) + 1], i & 31);
}

template <int DIN, int DOUT, int NV, class Count>
__global__ void __launch_bounds__(kLogitThreads, 5) logits_adjust_kernel(const __grid_constant__ LogitArgs a) {
  using In = LogitType<DIN>;
  using Out = LogitType<DOUT>;
  using TI = typename In::T;
  using TO = typename Out::T;
  constexpr int PER = 16 / (int)sizeof(TI), CHUNK = kLogitThreads * NV * PER;
  constexpr int WORDS = CHUNK / 32 + 2;
  constexpr uint32_t kPrompt = 1u << (8 * sizeof(Count) - 1);
  extern __shared__ __align__(16) uint32_t logit_smem[];
  Count* count = reinterpret_cast<Count*>(logit_smem);                      // [CHUNK]
  uint32_t* marks = logit_smem + CHUNK * sizeof(Count) / 4;                 // [WORDS] history or bias list
  uint32_t* bits = marks + WORDS;                                           // [WORDS] grammar
  uint32_t* list = bits + WORDS;                                            // marked tokens, then their values
  __shared__ unsigned long long s_best[kLogitThreads / 32];
  constexpr int kShort = 64;  // a chunk's biases that fit the short list
  __shared__ int s_listed, s_biases;
  __shared__ int s_bias_k[kShort];
  __shared__ float s_bias_v[kShort];
  const int m = blockIdx.y, c0 = blockIdx.x * CHUNK, len = min(CHUNK, a.V - c0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // ---- the chunk's logits: whole 16-byte pieces; up to PER - 1 values at either end
  const TI* x = reinterpret_cast<const TI*>(a.logits) + m * a.logits_row + c0;
  TO* y = reinterpret_cast<TO*>(a.out) + m * a.out_row + c0;
  const int head = min(len, (int)(((16u - ((uintptr_t)x & 15u)) & 15u) / sizeof(TI)));
  const int nvec = (len - head) / PER, tail = head + nvec * PER;
  uint4 v[NV];
#pragma unroll
  for (int j = 0; j < NV; j++)
    if (tid + j * kLogitThreads < nvec)
      v[j] = *(reinterpret_cast<const uint4*>(x + head) + tid + j * kLogitThreads);
  // thread t < head: value t; head <= t < head + len - tail: value tail + t - head
  const int edge = tid < head ? tid : tail + tid - head;
  float edge_x = 0.0f;
  if (edge < len && tid < 2 * PER) edge_x = In::get(x[edge]);
  // the first history entries do not wait for the length
  constexpr int HU = 4;
  const int* tok = a.history + m * a.history_row;
  int t[HU];
  const int* bt = a.bias_tokens + m * a.bias_row;
  const float* bv = a.bias_values + m * a.bias_row;
  int b_token = -1;
  float b_value = 0.0f;
  if (warp == 0 && lane < a.biases) {
    b_token = bt[lane];
    b_value = bv[lane];
  }
  if (a.history) {
#pragma unroll
    for (int u = 0; u < HU; u++) t[u] = tid + u * kLogitThreads < a.history_cap ? tok[tid + u * kLogitThreads] : -1;
  }

  // ---- mark and count
  const int hist = a.history ? min(max(a.history_lens[m], 0), a.history_cap) : 0;
  const int prompt = a.prompt_lens && hist > 0 ? a.prompt_lens[m] : 0;
  const bool any = hist > 0 || a.biases > 0;
  if (any) {
    for (int i = tid; i < (int)(CHUNK * sizeof(Count) / 16); i += kLogitThreads)
      reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
  }
  if (tid == 0) s_listed = 0;
  for (int i = tid; i < WORDS; i += kLogitThreads) {
    marks[i] = 0;
    if (a.allowed) bits[i] = (c0 >> 5) + i < (a.V + 31) / 32 ? a.allowed[m * a.allowed_row + (c0 >> 5) + i] : 0u;
  }
  __syncthreads();
  auto mark = [&](unsigned k) {
    const uint32_t bit = 1u << (k & 31);
    if (!(atomicOr(&marks[k >> 5], bit) & bit)) list[atomicAdd(&s_listed, 1)] = k;
  };
  for (int i = tid; i < hist; i += HU * kLogitThreads) {
    int next[HU];
#pragma unroll
    for (int u = 0; u < HU; u++) {
      const int k = i + (HU + u) * kLogitThreads;
      next[u] = k < hist ? tok[k] : -1;
    }
    // which of this thread's entries lie in the chunk: few do, so they are taken one
    // after the other instead of testing each position of the step warp-wide
    unsigned here = 0;
#pragma unroll
    for (int u = 0; u < HU; u++)
      here |= (i + u * kLogitThreads < hist && t[u] >= 0 && (unsigned)(t[u] - c0) < (unsigned)len ? 1u : 0u) << u;
    while (here) {
      const int u = __ffs(here) - 1;
      here &= here - 1;
      int token = t[0];
#pragma unroll
      for (int w = 1; w < HU; w++) token = u == w ? t[w] : token;
      const unsigned k = (unsigned)(token - c0);
      mark(k);
      const uint32_t add = i + u * kLogitThreads < prompt ? kPrompt : 1u;
      uint32_t* word = sizeof(Count) == 2 ? logit_smem + (k >> 1) : logit_smem + k;
      const uint32_t shifted = sizeof(Count) == 2 ? add << (16 * (k & 1)) : add;
      if (add == 1u) atomicAdd(word, shifted); else atomicOr(word, shifted);
    }
#pragma unroll
    for (int u = 0; u < HU; u++) t[u] = next[u];
  }
  if (warp == 0) {  // the chunk's biases, in order (the first kShort of them are kept)
    int nb = 0;
    for (int i0 = 0; i0 < a.biases; i0 += 32) {
      const int token = b_token;
      const float b = b_value;
      const int i = i0 + 32 + lane;
      b_token = i < a.biases ? bt[i] : -1;
      b_value = i < a.biases ? bv[i] : 0.0f;
      const bool mine = token >= c0 && token < c0 + len;
      const unsigned all = __ballot_sync(0xffffffffu, mine);
      if (mine) {
        mark((unsigned)(token - c0));
        const int at = nb + __popc(all & ((1u << lane) - 1u));
        if (at < kShort) {
          s_bias_k[at] = token - c0;
          s_bias_v[at] = b;
        }
      }
      nb += __popc(all);
    }
    if (lane == 0) s_biases = nb;
  }

  // ---- the marked tokens; count[k] becomes the place of token k's value
  if (any) {
    const float rep = a.repetition ? a.repetition[m] : 1.0f;
    const float freq = a.frequency ? a.frequency[m] : 0.0f;
    const float pres = a.presence ? a.presence[m] : 0.0f;
    __syncthreads();
    const int short_list = s_biases <= kShort ? s_biases : 0;
    for (int p = tid; p < s_listed; p += kLogitThreads) {
      const int k = (int)list[p];
      float z = In::get(x[k]);
      const uint32_t c = count[k], times = c & (kPrompt - 1u);
      if (c != 0) z = z > 0.0f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
      if (times != 0) z = __fsub_rn(__fsub_rn(z, __fmul_rn(freq, (float)times)), pres);
      for (int i = 0; i < short_list; i++)
        if (s_bias_k[i] == k) z = __fadd_rn(z, s_bias_v[i]);
      list[p] = __float_as_uint(z);
      count[k] = (Count)p;
    }
    __syncthreads();
  }
  if (a.biases > kShort && s_biases > kShort) {
    // too many to look through for every token: one warp adds them, 32 at a time, in
    // order; of equal tokens the lowest lane adds
    if (warp == 0) {
      for (int i0 = 0; i0 < a.biases; i0 += 32) {
        const int i = i0 + lane;
        const int token = i < a.biases ? bt[i] : -1;
        const float b = i < a.biases ? bv[i] : 0.0f;
        const bool mine = token >= c0 && token < c0 + len;
        if (!__any_sync(0xffffffffu, mine)) continue;
        const unsigned same = __match_any_sync(0xffffffffu, mine ? token : -1 - lane);
        uint32_t* at = &list[mine ? count[token - c0] : 0];
        float z = mine ? __uint_as_float(*at) : 0.0f;
        if (__all_sync(0xffffffffu, same == 1u << lane)) {
          z = __fadd_rn(z, b);
        } else {
          for (int l = 0; l < 32; l++) {
            const float other = __shfl_sync(0xffffffffu, b, l);
            if ((same >> l) & 1u) z = __fadd_rn(z, other);
          }
        }
        __syncwarp();
        if (mine && __ffs(same) - 1 == lane) *at = __float_as_uint(z);
        __syncwarp();
      }
    }
    __syncthreads();
  }
  auto marked = [&](int i) { return __uint_as_float(list[count[i]]); };

  // ---- stream
  float best = -INFINITY;
  int best_i = -1;
  float edge_z = -INFINITY;
  if (edge < len && tid < 2 * PER) {
    float z = edge_x;
    if ((marks[edge >> 5] >> (edge & 31)) & 1u) z = marked(edge);
    if (a.allowed && !((bits[edge >> 5] >> (edge & 31)) & 1u)) z = -INFINITY;
    edge_z = z;
    y[edge] = Out::put(z);
  }
  const bool wide = ((uintptr_t)(y + head) & 15u) == 0;
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int at = tid + j * kLogitThreads;
    if (at >= nvec) continue;
    const int i = head + at * PER;
    const uint32_t mk = bits_from(marks, i), ok = a.allowed ? bits_from(bits, i) : 0xffffffffu;
    const TI* e = reinterpret_cast<const TI*>(&v[j]);
    float z[PER];
#pragma unroll
    for (int u = 0; u < PER; u++) z[u] = In::get(e[u]);
    if (mk & ((1u << PER) - 1u)) {
#pragma unroll
      for (int u = 0; u < PER; u++)
        if ((mk >> u) & 1u) z[u] = marked(i + u);
    }
    float top = -INFINITY;  // (fmaxf passes a NaN over)
#pragma unroll
    for (int u = 0; u < PER; u++) {
      if (!((ok >> u) & 1u)) z[u] = -INFINITY;
      top = fmaxf(top, z[u]);
    }
    if (top > best) {
      best = top;
#pragma unroll
      for (int u = PER - 1; u >= 0; u--)
        if (z[u] == top) best_i = i + u;
    }
    if (wide) {
      alignas(16) TO r[PER];
#pragma unroll
      for (int u = 0; u < PER; u++) r[u] = Out::put(z[u]);
#pragma unroll
      for (int u = 0; u < PER * (int)sizeof(TO) / 16; u++)
        __stcs(reinterpret_cast<uint4*>(y + i) + u, reinterpret_cast<const uint4*>(r)[u]);
    } else {
#pragma unroll
      for (int u = 0; u < PER; u++) y[i + u] = Out::put(z[u]);
    }
  }

  if (!a.token) return;
  // equal values are settled by the key's index part: the lowest index has the largest
  auto key = [&](float z, int i) {
    return z > -INFINITY ? ((unsigned long long)logit_order(z) << 32) | (0xffffffffu - (uint32_t)(c0 + i)) : 0ull;
  };
  unsigned long long k = key(best, best_i);
  const unsigned long long ek = key(edge_z, edge);
  k = ek > k ? ek : k;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long p = __shfl_xor_sync(0xffffffffu, k, o);
    k = p > k ? p : k;
  }
  if (lane == 0) s_best[warp] = k;
  __syncthreads();
  if (tid != 0) return;
  for (int w = 1; w < kLogitThreads / 32; w++) k = s_best[w] > k ? s_best[w] : k;
  if (gridDim.x > 1) {
    if (k != 0) atomicMax(a.best + m, k);
    __threadfence();
    if (atomicAdd(a.arrived + m, 1u) != gridDim.x - 1) return;
    __threadfence();
    k = atomicExch(a.best + m, 0ull);
    a.arrived[m] = 0;
  }
  a.token[m] = k == 0 ? -1 : (int)(0xffffffffu - (uint32_t)k);
}

// ------------------------------------------------------------------ host side
size_t logits_workspace_bytes(int M) { return (size_t)M * (sizeof(unsigned long long) + sizeof(unsigned)); }

template <int DIN, int DOUT, int NV, class Count>
static cudaError_t launch_logits_n(const LogitArgs& a, cudaStream_t st) {
  constexpr int CHUNK = kLogitThreads * NV * 16 / (int)sizeof(typename LogitType<DIN>::T);
  constexpr int kFixed = CHUNK * (int)sizeof(Count) + 2 * (CHUNK / 32 + 2) * (int)sizeof(uint32_t);
  constexpr auto kern = logits_adjust_kernel<DIN, DOUT, NV, Count>;
  if (kFixed + CHUNK * 4 > 48 * 1024)
    if (cudaError_t e = allow_smem<kern>(kFixed + CHUNK * 4)) return e;
  // a chunk's marked tokens: no more than it has, and no more than entries that mark
  const long long entries = (long long)(a.history ? a.history_cap : 0) + a.biases;
  const int smem = kFixed + (int)(entries < CHUNK ? entries : CHUNK) * 4;
  kern<<<dim3((unsigned)((a.V + CHUNK - 1) / CHUNK), (unsigned)a.M), kLogitThreads, smem, st>>>(a);
  return cudaGetLastError();
}

// The largest chunk (4, 2 or 1 16-byte loads per thread) that still gives every SM
// two CTAs: more loads in flight per CTA and fewer readings of the history against
// idle SMs.  Histories that a 15-bit count cannot hold take 31-bit ones.
template <int DIN, int DOUT>
static cudaError_t launch_logits_t(const LogitArgs& a, cudaStream_t st) {
  const long long per = kLogitThreads * 16 / (int)sizeof(typename LogitType<DIN>::T);
  auto ctas = [&](int nv) { return (a.V + per * nv - 1) / (per * nv) * a.M; };
  if (a.history && a.history_cap > 32767) return launch_logits_n<DIN, DOUT, 2, uint32_t>(a, st);
  if (ctas(4) >= 2 * sm_count()) return launch_logits_n<DIN, DOUT, 4, uint16_t>(a, st);
  if (ctas(2) >= 2 * sm_count()) return launch_logits_n<DIN, DOUT, 2, uint16_t>(a, st);
  return launch_logits_n<DIN, DOUT, 1, uint16_t>(a, st);
}

cudaError_t launch_logits_adjust(LogitArgs a, int din, int dout, void* ws, cudaStream_t st) {
  a.best = (unsigned long long*)ws;
  a.arrived = ws ? (unsigned*)(a.best + a.M) : nullptr;
  if (din == 0) return launch_logits_t<0, 0>(a, st);
  if (din == 1) return dout == 1 ? launch_logits_t<1, 1>(a, st) : launch_logits_t<1, 0>(a, st);
  return dout == 2 ? launch_logits_t<2, 2>(a, st) : launch_logits_t<2, 0>(a, st);
}

}  // namespace aria_q4
