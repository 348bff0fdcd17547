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
// One pass over the logits: a CTA takes a chunk of one row, counts the history's
// tokens that fall into it in shared memory (one word per token: bit 31 = in the
// prompt, the rest = times generated; integer atomics, so any order gives the same
// counts), adds up its biases, then streams the chunk with 16-byte accesses.  The
// largest value is joined over a row's CTAs by a 64-bit maximum of (ordered value,
// ~index) and a counter; the last CTA writes the token and clears both.  Bound: HBM,
// 2 e bytes per logit + 1/8 for the mask; small calls by their launch.
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

template <int DIN, int DOUT>
__global__ void __launch_bounds__(kLogitThreads) logits_adjust_kernel(const LogitArgs a) {
  using In = LogitType<DIN>;
  using Out = LogitType<DOUT>;
  using TI = typename In::T;
  using TO = typename Out::T;
  extern __shared__ uint32_t logit_smem[];
  uint32_t* count = logit_smem;                                    // [chunk]
  float* bias = reinterpret_cast<float*>(logit_smem + a.chunk);    // [chunk] with biases
  uint32_t* bits = logit_smem + (a.bias_tokens ? 2 : 1) * a.chunk;  // [chunk / 32 + 2] with a mask
  __shared__ unsigned long long s_best[kLogitThreads / 32];
  const int m = blockIdx.y, c0 = blockIdx.x * a.chunk, c1 = min(a.V, c0 + a.chunk), len = c1 - c0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  for (int i = tid; i < len; i += kLogitThreads) {
    count[i] = 0;
    if (a.bias_tokens) bias[i] = 0.0f;
  }
  if (a.allowed)  // c0 is a multiple of 32
    for (int i = tid; i < (len + 31) / 32 + 1; i += kLogitThreads)
      bits[i] = (c0 >> 5) + i < (a.V + 31) / 32 ? a.allowed[m * a.allowed_row + (c0 >> 5) + i] : 0u;
  __syncthreads();
  const int hist = a.history ? min(max(a.history_lens[m], 0), a.history_cap) : 0;
  const int prompt = a.prompt_lens && hist > 0 ? a.prompt_lens[m] : 0;
  const int* tok = a.history + m * a.history_row;
  for (int i = tid; i < hist; i += kLogitThreads) {
    const int v = tok[i] - c0;
    if (tok[i] >= 0 && v >= 0 && v < len) {
      if (i < prompt) atomicOr(&count[v], 0x80000000u); else atomicAdd(&count[v], 1u);
    }
  }
  if (a.bias_tokens && warp == 0) {
    // 32 entries at a time, in order; the lowest lane of equal tokens adds them up
    for (int i0 = 0; i0 < a.biases; i0 += 32) {
      const int i = i0 + lane;
      const int v = i < a.biases ? a.bias_tokens[m * a.bias_row + i] : -1;
      const float b = i < a.biases ? a.bias_values[m * a.bias_row + i] : 0.0f;
      const unsigned same = __match_any_sync(0xffffffffu, v);
      const bool mine = v >= c0 && v < c1;
      float s = mine ? bias[v - c0] : 0.0f;
      for (int l = 0; l < 32; l++) {
        const float x = __shfl_sync(0xffffffffu, b, l);
        if ((same >> l) & 1u) s += x;
      }
      if (mine && (__ffs(same) - 1) == lane) bias[v - c0] = s;
      __syncwarp();
    }
  }
  __syncthreads();

  const float rep = a.repetition ? a.repetition[m] : 1.0f;
  const float freq = a.frequency ? a.frequency[m] : 0.0f;
  const float pres = a.presence ? a.presence[m] : 0.0f;
  const TI* x = reinterpret_cast<const TI*>(a.logits) + m * a.logits_row + c0;
  TO* y = reinterpret_cast<TO*>(a.out) + m * a.out_row + c0;
  float best = -INFINITY;
  int best_i = -1;
  auto one = [&](int i, float v) {
    const uint32_t c = count[i];
    if (c != 0) {
      v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      const uint32_t times = c & 0x7fffffffu;
      if (times != 0) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)times)), pres);
    }
    if (a.bias_tokens) v = __fadd_rn(v, bias[i]);
    if (a.allowed && !((bits[i >> 5] >> (i & 31)) & 1u)) v = -INFINITY;
    if (v > best) {
      best = v;
      best_i = i;
    }
    return v;
  };
  // 16-byte accesses where both rows start at the same distance from a 16-byte
  // boundary (equal types), single values at the ends and otherwise
  constexpr int PER = 16 / (int)sizeof(TI);
  const int head_x = (int)(((16u - ((uintptr_t)x & 15u)) & 15u) / sizeof(TI));
  const bool vec = DIN == DOUT && ((uintptr_t)x & 15u) == ((uintptr_t)y & 15u);
  const int head = vec ? min(head_x, len) : len;
  const int nvec = (len - head) / PER;
  for (int i = tid; i < head; i += kLogitThreads) y[i] = Out::put(one(i, In::get(x[i])));
  for (int j = tid; j < nvec; j += kLogitThreads) {
    uint4 w = *reinterpret_cast<const uint4*>(x + head + j * PER);
    TI* e = reinterpret_cast<TI*>(&w);
#pragma unroll
    for (int u = 0; u < PER; u++) {
      const TO r = Out::put(one(head + j * PER + u, In::get(e[u])));
      e[u] = *reinterpret_cast<const TI*>(&r);
    }
    *reinterpret_cast<uint4*>(y + head + j * PER) = w;
  }
  for (int i = head + nvec * PER + tid; i < len; i += kLogitThreads) y[i] = Out::put(one(i, In::get(x[i])));

  if (!a.token) return;
  unsigned long long k =
      best_i < 0 ? 0ull
                 : ((unsigned long long)logit_order(best) << 32) | (0xffffffffu - (uint32_t)(c0 + best_i));
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

template <int DIN, int DOUT>
static cudaError_t launch_logits_t(const LogitArgs& a, size_t smem, cudaStream_t st) {
  auto kern = logits_adjust_kernel<DIN, DOUT>;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kern<<<dim3((unsigned)((a.V + a.chunk - 1) / a.chunk), (unsigned)a.M), kLogitThreads, smem, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_logits_adjust(LogitArgs a, int din, int dout, void* ws, cudaStream_t st) {
  a.best = (unsigned long long*)ws;
  a.arrived = ws ? (unsigned*)(a.best + a.M) : nullptr;
  const int sms = sm_count();
  // chunks of 1024 to 8192 tokens: the largest that still gives every SM two
  int chunk = 8192;
  while (chunk > 1024 && (long long)((a.V + chunk - 1) / chunk) * a.M < 2LL * sms) chunk /= 2;
  a.chunk = chunk;
  const size_t smem = ((size_t)chunk * (a.bias_tokens ? 2 : 1) + chunk / 32 + 2) * sizeof(uint32_t);
  if (din == 0) return launch_logits_t<0, 0>(a, smem, st);
  if (din == 1) return dout == 1 ? launch_logits_t<1, 1>(a, smem, st) : launch_logits_t<1, 0>(a, smem, st);
  return dout == 2 ? launch_logits_t<2, 2>(a, smem, st) : launch_logits_t<2, 0>(a, smem, st);
}

}  // namespace aria_q4
