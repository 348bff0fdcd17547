// cache_evict.cu -- eviction from a paged KV cache by accumulated attention weight.
//
// Every (sequence, key/value head) row of n > keep slots keeps `keep` of them: the
// newest `recent` positions and the first `sinks` ones, then those of the largest
// weight, ties to the lowest slot (NaN counts as the lowest weight).  The i-th
// survivor at a slot >= keep moves into the i-th slot < keep that is given up, K and
// V rows, weight and position with it, so a row that gives up one slot moves one row
// and not the cache, and no row that is read is written.  Slots keep .. n - 1 end
// with weight 0 and position -1.
//
// One thread-block cluster of 1 to 8 CTAs per row.  A weight becomes an unsigned key
// of the same order (kept positions: the largest key); the keep-th largest key is
// found by three counting passes over 11, 11 and 10 bits with the keys in shared
// memory, the CTAs' counts added over distributed shared memory; block and cluster
// prefix sums then rank ties, holes and movers, so the result does not depend on
// timing.  What the operator cannot do without is 16 bytes per slot (weight and
// position, read and written) and 2 x 2 rows per moved slot.
#include "q4_common.cuh"
#include "q4_paged.cuh"
#include "q4_status.cuh"

namespace aria_q4 {

constexpr int kEvictThreads = 256;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictBins = 2048;
constexpr int kEvictHistBytes = 2 * kEvictBins * (int)sizeof(uint32_t);
constexpr int kEvictMaxCluster = 8;
constexpr int kEvictKeys = 40 * 1024;  // keys a CTA can hold in shared memory (160 KB)

// order-preserving: a < b <=> key(a) < key(b); -0 = +0; NaN below everything
__device__ __forceinline__ uint32_t evict_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t ld_dsmem_u32(const uint32_t* local, uint32_t rank) {
  uint32_t remote, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(tc_smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}

// exclusive prefix sum over the block's threads of (x, y); totals in tx, ty
__device__ __forceinline__ void block_scan2(uint32_t& x, uint32_t& y, uint32_t& tx, uint32_t& ty,
                                            uint32_t (*ws)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t ix = x, iy = y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t ax = __shfl_up_sync(0xffffffffu, ix, o), ay = __shfl_up_sync(0xffffffffu, iy, o);
    if (lane >= o) {
      ix += ax;
      iy += ay;
    }
  }
  __syncthreads();  // ws may still be read by a previous scan
  if (lane == 31) {
    ws[warp][0] = ix;
    ws[warp][1] = iy;
  }
  __syncthreads();
  uint32_t bx = 0, by = 0;
  tx = ty = 0;
#pragma unroll
  for (int w = 0; w < kEvictWarps; w++) {
    const uint32_t a = ws[w][0], b = ws[w][1];
    if (w < warp) {
      bx += a;
      by += b;
    }
    tx += a;
    ty += b;
  }
  x = bx + ix - x;
  y = by + iy - y;
}

template <bool SMEM_KEYS>
__global__ void __launch_bounds__(kEvictThreads, 4) cache_evict_kernel(const EvictArgs a) {
  extern __shared__ uint32_t evict_smem[];
  uint32_t* hist = evict_smem;                      // [2][kEvictBins]
  uint32_t* keys = evict_smem + 2 * kEvictBins;     // this CTA's slots
  __shared__ uint32_t ws[kEvictWarps][2];
  __shared__ uint32_t counts[4];                    // read by the other CTAs of the cluster
  __shared__ uint32_t s_bin, s_above;
  const int tid = threadIdx.x;
  const int cs = a.cluster;
  const uint32_t rank = cs > 1 ? blockIdx.x % cs : 0;
  const int row = blockIdx.x / cs, m = row / a.Hkv, hk = row % a.Hkv;
  auto cluster_sync = [&]() {
    if (cs > 1) cluster_sync_all(); else __syncthreads();
  };
  auto peer = [&](const uint32_t* p, uint32_t r) { return cs > 1 ? ld_dsmem_u32(p, r) : *p; };

  const int n = (int)min((long long)max(a.lens[m], 0), a.slots);
  const size_t at = (size_t)row * a.cap;
  const float* win = a.weights_in + at;
  const int* pin = a.pos_in + at;
  float* wout = a.weights_out + at;
  int* pout = a.pos_out + at;
  if (hk == 0 && rank == 0 && tid == 0 && a.lens_out) a.lens_out[m] = min(n, a.keep);

  // this CTA's slots [b, e), and per thread an odd number of consecutive ones
  // (odd: the threads' shared-memory reads then fall into different banks)
  const int share = (n + cs - 1) / cs;
  const int b = min(n, (int)rank * share), e = min(n, b + share);
  const bool copy_w = wout != win, copy_p = pout != pin;
  if (n <= a.keep) {  // nothing to give up (the whole cluster returns)
    for (int i = b + tid; i < e; i += kEvictThreads) {
      if (copy_w) wout[i] = win[i];
      if (copy_p) pout[i] = pin[i];
    }
    return;
  }
  const int newest = a.next_pos[m] - a.recent;
  auto make_key = [&](int i) {
    const int p = pin[i];
    return p >= newest || p < a.sinks ? 0xffffffffu : evict_key(win[i]);
  };
  auto key = [&](int i) { return SMEM_KEYS ? keys[i - b] : make_key(i); };

  for (int i = tid; i < 2 * kEvictBins; i += kEvictThreads) hist[i] = 0;
  if (SMEM_KEYS || copy_w || copy_p)
    for (int i = b + tid; i < e; i += kEvictThreads) {
      // (outputs of their own get what stays where it is here; holes are overwritten below)
      const int p = pin[i];
      const float w = win[i];
      if (SMEM_KEYS) keys[i - b] = p >= newest || p < a.sinks ? 0xffffffffu : evict_key(w);
      if (copy_w) wout[i] = i < a.keep ? w : 0.0f;
      if (copy_p) pout[i] = i < a.keep ? p : -1;
    }
  __syncthreads();

  // ---- the keep-th largest key T, and how many slots with exactly T are kept
  uint32_t prefix = 0, need = (uint32_t)a.keep;
#pragma unroll
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bmask = pass == 2 ? 1023u : 2047u;
    const int up = pass == 0 ? 32 : pass == 1 ? 21 : 10;  // bits above are settled
    uint32_t* h = hist + (pass & 1) * kEvictBins;
    for (int i = b + tid; i < e; i += kEvictThreads) {
      const uint32_t k = key(i);
      if (pass == 0 || (k >> up) == (prefix >> up)) atomicAdd(&h[(k >> shift) & bmask], 1u);
    }
    cluster_sync();
    // thread t: bins 2047 - BPT t - (0 .. BPT - 1), from the largest key down
    constexpr int BPT = kEvictBins / kEvictThreads;
    uint32_t cnt[BPT], sum = 0;
#pragma unroll
    for (int u = 0; u < BPT; u++) {
      const int bin = kEvictBins - 1 - BPT * tid - u;
      cnt[u] = 0;
      for (int r = 0; r < cs; r++) cnt[u] += peer(&h[bin], (uint32_t)r);
      sum += cnt[u];
    }
    uint32_t before = sum, zero = 0, t0, t1;
    block_scan2(before, zero, t0, t1, ws);
#pragma unroll
    for (int u = 0; u < BPT; u++) {
      if (before < need && before + cnt[u] >= need) {
        s_bin = (uint32_t)(kEvictBins - 1 - BPT * tid - u);
        s_above = before;
      }
      before += cnt[u];
    }
    // the first pass's counts, which every CTA read before this pass's barrier
    if (pass == 1)
      for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[i] = 0;
    __syncthreads();
    prefix |= s_bin << shift;
    need -= s_above;
  }
  const uint32_t T = prefix;

  // ---- ties with T are kept lowest slot first: rank them
  const int items = ((share + kEvictThreads - 1) / kEvictThreads) | 1;
  const int i0 = min(e, b + tid * items), i1 = min(e, i0 + items);
  uint32_t ties = 0, none = 0, tot_ties, tot_none;
  for (int i = i0; i < i1; i++) ties += key(i) == T;
  block_scan2(ties, none, tot_ties, tot_none, ws);
  if (tid == 0) counts[0] = tot_ties;
  cluster_sync();
  for (uint32_t r = 0; r < rank; r++) ties += peer(&counts[0], r);

  // ---- holes below keep and survivors that have to move: rank them
  uint32_t holes = 0, movers = 0, tot_h, tot_m;
  uint32_t tie = ties;
  for (int i = i0; i < i1; i++) {
    const uint32_t k = key(i);
    const bool kept = k > T || (k == T && tie++ < need);
    holes += !kept && i < a.keep;
    movers += kept && i >= a.keep;
  }
  block_scan2(holes, movers, tot_h, tot_m, ws);
  if (tid == 0) {
    counts[1] = tot_h;
    counts[2] = tot_m;
  }
  cluster_sync();
  uint32_t all = 0;
  for (uint32_t r = 0; r < (uint32_t)cs; r++) {
    const uint32_t ch = peer(&counts[1], r), cm = peer(&counts[2], r);
    if (r < rank) {
      holes += ch;
      movers += cm;
    }
    all += ch;
  }
  int* to = a.lists + (size_t)row * 2 * a.list_len;
  int* from = to + a.list_len;
  tie = ties;
  for (int i = i0; i < i1; i++) {
    const uint32_t k = key(i);
    const bool kept = k > T || (k == T && tie++ < need);
    if (i < a.keep && !kept) to[holes++] = i;
    if (i >= a.keep && kept) from[movers++] = i;
  }
  cluster_sync();  // the lists are complete, and no key is read any more

  // ---- move weights and positions, then K and V rows
  for (int i = (int)rank * kEvictThreads + tid; i < (int)all; i += cs * kEvictThreads) {
    const int d = __ldcg(to + i), s = __ldcg(from + i);
    wout[d] = win[s];
    pout[d] = pin[s];
  }
  const int cpr = a.row_bytes >> 4;  // 16-byte chunks per row (a power of two)
  const int rows_per_step = kEvictThreads / cpr;
  const int ch = tid % cpr, r0 = tid / cpr;
  const int step = cs * rows_per_step;
  auto row_of = [&](int slot) -> long long {
    const int page = a.table[(long long)m * a.table_stride + slot / a.page_size];
    if (page < 0 || page >= a.num_pages) return -1;
    return (long long)page * a.page_stride + (long long)(slot % a.page_size) * a.slot_stride +
           (long long)hk * a.head_stride + ch * 8;
  };
  constexpr int U = 4;
  for (int i = (int)rank * rows_per_step + r0; i < (int)all; i += U * step) {
    long long src[U], dst[U];
    uint4 kv[U], vv[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      src[u] = dst[u] = -1;
      if (i + u * step < (int)all) {
        src[u] = row_of(__ldcg(from + i + u * step));
        dst[u] = row_of(__ldcg(to + i + u * step));
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (src[u] >= 0 && dst[u] >= 0) {
        kv[u] = *reinterpret_cast<const uint4*>(a.k_pages + src[u]);
        vv[u] = *reinterpret_cast<const uint4*>(a.v_pages + src[u]);
      }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (src[u] >= 0 && dst[u] >= 0) {
        *reinterpret_cast<uint4*>(a.k_pages + dst[u]) = kv[u];
        *reinterpret_cast<uint4*>(a.v_pages + dst[u]) = vv[u];
      }
  }
  cluster_sync();  // the moved weights have been read; no CTA reads another's memory any more
  for (int i = max(b, a.keep) + tid; i < e; i += kEvictThreads) {
    if (!copy_w) wout[i] = 0.0f;
    if (!copy_p) pout[i] = -1;
  }
}

// ------------------------------------------------------------------ host side
static long long evict_list_len(long long slots, int keep) {
  const long long rest = slots - keep;
  return rest <= 0 ? 0 : (rest < keep ? rest : keep);
}

size_t evict_workspace_bytes(int M, int Hkv, long long slots, int keep) {
  return (size_t)M * Hkv * 2 * evict_list_len(slots, keep) * sizeof(int);
}

template <bool SMEM_KEYS>
static cudaError_t launch_evict_t(const EvictArgs& a, size_t smem, cudaStream_t st) {
  constexpr auto kern = cache_evict_kernel<SMEM_KEYS>;
  if (cudaError_t e = allow_smem<kern>(kEvictHistBytes + kEvictKeys * (int)sizeof(uint32_t))) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.M * a.Hkv * a.cluster));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

cudaError_t launch_cache_evict(EvictArgs a, void* ws, cudaStream_t st) {
  a.lists = (int*)ws;
  a.list_len = evict_list_len(a.slots, a.keep);
  const int sms = sm_count();
  const int rows = a.M * a.Hkv;
  a.cluster = kEvictMaxCluster;
  while (a.cluster > 1 && ((long long)rows * a.cluster > 2 * sms || a.slots / a.cluster < 1024)) a.cluster /= 2;
  const long long share = (a.slots + a.cluster - 1) / a.cluster;
  if (share <= kEvictKeys) return launch_evict_t<true>(a, kEvictHistBytes + (size_t)share * sizeof(uint32_t), st);
  return launch_evict_t<false>(a, kEvictHistBytes, st);
}

}  // namespace aria_q4
