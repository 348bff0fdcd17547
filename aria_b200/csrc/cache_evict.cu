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
// Choosing: one thread-block cluster of 1 to 8 CTAs per row.  A weight becomes an
// unsigned key of the same order (kept positions: the largest key); the keep-th largest
// key is found by up to three counting passes over 11, 11 and 10 bits with the keys in
// shared memory, the CTAs' counts added over distributed shared memory, ending as soon
// as a bin is taken whole.  Ballots and prefix sums over warps, block and cluster then
// rank ties, holes and movers, so the result does not depend on timing.
// Moving: rows are small (64 to 512 bytes) and scattered, so what counts is how many
// are under way.  Where a row can give up more than kEvictFused slots a second kernel
// spreads all rows' moves over all SMs (one CTA moves about 34 bytes a cycle each way,
// an SM's share of HBM is 23: in one kernel the SMs that chose fewer rows stood idle,
// 140 us instead of 133 for 64 x 14 rows of up to 8191 slots cut to 4096, 72 instead of
// 51 for 16 x 14); a few slots
// are moved where they were chosen, which saves a launch.
// What the operator cannot do without is 16 bytes per slot (weight and position, read
// and written) and 2 x 2 rows per moved slot.
#include <algorithm>

#include "q4_common.cuh"
#include "q4_paged.cuh"
#include "q4_status.cuh"

namespace aria_q4 {

constexpr int kEvictBins = 2048;
constexpr int kEvictHistBytes = 2 * kEvictBins * (int)sizeof(uint32_t);
constexpr int kEvictMaxCluster = 8;
constexpr int kEvictFused = 64;  // slots a row can give up without a second kernel
constexpr int kEvictKeys = 40 * 1024;  // keys a CTA can hold in shared memory (160 KB)
constexpr int kEvictMaxSmem = 224 * 1024;

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

__device__ __forceinline__ uint4 ld_dsmem_u4(const uint32_t* local, uint32_t rank) {
  uint32_t remote;
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(tc_smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

// The rows of the moves [first, end) of a row's lists, by a block of THREADS: the rows'
// places are worked out for up to kEvictBatch moves at a time (offs: shared memory for
// two per move), so that the copies wait for nothing but their own data; 16 bytes of K
// and of V per thread and step, 4 steps at a time.
constexpr int kEvictBatch = 256;
template <int THREADS>
__device__ __forceinline__ void evict_move(const EvictArgs& a, int m, int hk, const int* to, const int* from, int first,
                                           int end, long long* offs) {
  const int tid = threadIdx.x;
  const int cpr = a.row_bytes >> 4;  // 16-byte chunks per row (a power of two)
  const int step = THREADS / cpr, ch = tid % cpr, r0 = tid / cpr;
  const int* table = a.table + (long long)m * a.table_stride;
  auto row_of = [&](int slot) -> long long {
    const int pi = (int)(((unsigned long long)(unsigned)slot * a.page_mul) >> a.page_shift);
    const int page = table[pi];
    if (page < 0 || page >= a.num_pages) return -1;
    return (long long)page * a.page_stride + (long long)(slot - pi * a.page_size) * a.slot_stride +
           (long long)hk * a.head_stride;
  };
  for (int base = first; base < end; base += kEvictBatch) {
    const int cnt = min(kEvictBatch, end - base);
    __syncthreads();
    for (int i = tid; i < 2 * cnt; i += THREADS)
      offs[i] = row_of(i < cnt ? __ldcg(from + base + i) : __ldcg(to + base + i - cnt));
    __syncthreads();
    constexpr int U = 4;
    for (int i = r0; i < cnt; i += U * step) {
      long long dst[U];
      uint4 kv[U], vv[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int at = i + u * step;
        dst[u] = -1;
        if (at < cnt && offs[at] >= 0 && offs[cnt + at] >= 0) {
          const long long src = offs[at] + ch * 8;
          dst[u] = offs[cnt + at] + ch * 8;
          kv[u] = *reinterpret_cast<const uint4*>(a.k_pages + src);
          vv[u] = *reinterpret_cast<const uint4*>(a.v_pages + src);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (dst[u] >= 0) {
          *reinterpret_cast<uint4*>(a.k_pages + dst[u]) = kv[u];
          *reinterpret_cast<uint4*>(a.v_pages + dst[u]) = vv[u];
        }
    }
  }
}

// SMEM_KEYS: keys in shared memory; otherwise they are formed again at every pass
template <bool SMEM_KEYS, int kEvictThreads>
__global__ void __launch_bounds__(kEvictThreads, 1024 / kEvictThreads) cache_evict_kernel(
    const __grid_constant__ EvictArgs a) {
  constexpr int kEvictWarps = kEvictThreads / 32;
  extern __shared__ __align__(16) uint32_t evict_smem[];
  uint32_t* hist = evict_smem;                      // [2][kEvictBins]
  uint32_t* kept_bits = evict_smem + 2 * kEvictBins;  // [share / 32 + 1]
  uint32_t* keys = kept_bits + a.bit_words;           // this CTA's slots, then its row's lists
  __shared__ uint32_t ws[kEvictWarps][2];
  __shared__ uint32_t counts[4];                    // read by the other CTAs of the cluster
  __shared__ uint32_t s_bin, s_above, s_in;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t lt = (1u << lane) - 1u;
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

  // this CTA's slots [b, e) and this warp's [wb, we): whole groups of 32
  const int share = ((n + cs - 1) / cs + 31) & ~31;
  const int b = min(n, (int)rank * share), e = min(n, b + share);
  const int wshare = ((share + kEvictWarps - 1) / kEvictWarps + 31) & ~31;
  const int wb = min(e, b + warp * wshare), we = min(e, wb + wshare);
  const bool copy_w = wout != win, copy_p = pout != pin;
  if (!a.fused) grid_dep_launch();
  if (n <= a.keep) {  // nothing to give up (the whole cluster returns)
    if (!a.fused && rank == 0 && tid == 0) a.moves[row] = 0;
    for (int i = b + tid; i < e; i += kEvictThreads) {
      if (copy_w) wout[i] = win[i];
      if (copy_p) pout[i] = pin[i];
    }
    return;
  }
  const int newest = a.next_pos[m] - a.recent;
  auto make_key = [&](float w, int p) { return p >= newest || p < a.sinks ? 0xffffffffu : evict_key(w); };
  auto key = [&](int i) { return SMEM_KEYS ? keys[i - b] : make_key(win[i], pin[i]); };

  for (int i = tid; i < 2 * kEvictBins / 4; i += kEvictThreads)
    reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  {
    constexpr int U = 8;
    for (int i0 = b + tid; i0 < e; i0 += U * kEvictThreads) {
      int p[U];
      float w[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = min(i0 + u * kEvictThreads, e - 1);
        p[u] = pin[i];
        w[u] = win[i];
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + u * kEvictThreads;
        if (i >= e) break;
        const uint32_t k = make_key(w[u], p[u]);
        if (SMEM_KEYS) keys[i - b] = k;
        atomicAdd(&hist[k >> 21], 1u);  // the first pass's counts
        // outputs of their own get here what stays where it is; holes are overwritten below
        if (copy_w) wout[i] = i < a.keep ? w[u] : 0.0f;
        if (copy_p) pout[i] = i < a.keep ? p[u] : -1;
      }
    }
  }

  // ---- the keep-th largest key T, and how many slots with exactly T are kept
  uint32_t T = 0, need = (uint32_t)a.keep;
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bmask = pass == 2 ? 1023u : 2047u;
    const int up = pass == 1 ? 21 : 10;  // bits above are settled (passes 1 and 2)
    uint32_t* h = hist + (pass & 1) * kEvictBins;
    if (pass > 0)
      for (int i = b + tid; i < e; i += kEvictThreads) {
        const uint32_t k = key(i);
        if ((k >> up) == (T >> up)) atomicAdd(&h[(k >> shift) & bmask], 1u);
      }
    cluster_sync();
    // thread t: bins 2047 - BPT t - (0 .. BPT - 1), from the largest key down
    constexpr int BPT = kEvictBins / kEvictThreads;
    const int top = kEvictBins - BPT * (tid + 1);
    uint32_t cnt[BPT] = {};  // cnt[u]: bin top + u
    if (BPT % 4 == 0) {
      for (int r = 0; r < cs; r++)
#pragma unroll
        for (int u = 0; u < BPT; u += 4) {
          const uint4 c = cs > 1 ? ld_dsmem_u4(h + top + u, r) : *reinterpret_cast<const uint4*>(h + top + u);
          cnt[u % BPT] += c.x;
          cnt[(u + 1) % BPT] += c.y;
          cnt[(u + 2) % BPT] += c.z;
          cnt[(u + 3) % BPT] += c.w;
        }
    } else {
      for (int r = 0; r < cs; r++)
#pragma unroll
        for (int u = 0; u < BPT; u++) cnt[u] += peer(h + top + u, (uint32_t)r);
    }
    uint32_t sum = 0;
#pragma unroll
    for (int u = 0; u < BPT; u++) sum += cnt[u];
    uint32_t before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t p = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += p;
    }
    if (lane == 31) ws[warp][0] = before;
    before -= sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kEvictWarps; w++)
      if (w < warp) before += ws[w][0];
    if (before < need && before + sum >= need) {
#pragma unroll
      for (int u = BPT - 1; u >= 0; u--) {
        if (before < need && before + cnt[u] >= need) {
          s_bin = (uint32_t)(top + u);
          s_above = before;
          s_in = cnt[u];
        }
        before += cnt[u];
      }
    }
    // the first pass's counts, which every CTA read before this pass's barrier
    if (pass == 1)
      for (int i = tid; i < kEvictBins / 4; i += kEvictThreads)
        reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    T |= s_bin << shift;
    need -= s_above;
    if (s_in == need) {  // the whole bin is kept: every key >= T
      need = 0xffffffffu;
      break;
    }
  }

  // sums over the warps before this one, and over the block, of two counts per warp
  auto block_prefix = [&](uint32_t& x, uint32_t& y, uint32_t& tx, uint32_t& ty) {
    __syncthreads();  // ws may still be read
    if (lane == 0) {
      ws[warp][0] = x;
      ws[warp][1] = y;
    }
    __syncthreads();
    x = y = tx = ty = 0;
#pragma unroll
    for (int w = 0; w < kEvictWarps; w++) {
      if (w < warp) {
        x += ws[w][0];
        y += ws[w][1];
      }
      tx += ws[w][0];
      ty += ws[w][1];
    }
  };

  // ---- ties with T are kept lowest slot first: rank them
  uint32_t ties = 0, none = 0, tot_ties, tot_none;
  if (need != 0xffffffffu) {
    for (int i0 = wb; i0 < we; i0 += 32)
      ties += __popc(__ballot_sync(0xffffffffu, i0 + lane < we && key(i0 + lane) == T));
    block_prefix(ties, none, tot_ties, tot_none);
    if (tid == 0) counts[0] = tot_ties;
    cluster_sync();
    for (uint32_t r = 0; r < rank; r++) ties += peer(&counts[0], r);
  }

  // ---- what is kept, as bits; holes below keep and survivors that have to move
  uint32_t holes = 0, movers = 0, tot_h, tot_m;
  for (int i0 = wb; i0 < we; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t k = i < we ? key(i) : 0u;
    const uint32_t eq = __ballot_sync(0xffffffffu, i < we && k == T);
    const uint32_t kept =
        __ballot_sync(0xffffffffu, i < we && (k > T || (k == T && ties + __popc(eq & lt) < need)));
    const uint32_t in = __ballot_sync(0xffffffffu, i < we), below = __ballot_sync(0xffffffffu, i < a.keep);
    ties += __popc(eq);
    holes += __popc(in & below & ~kept);
    movers += __popc(kept & ~below);
    if (lane == 0) kept_bits[(i0 - b) >> 5] = kept;
  }
  block_prefix(holes, movers, tot_h, tot_m);
  if (tid == 0) {
    counts[1] = tot_h;
    counts[2] = tot_m;
  }
  cluster_sync();  // (the keys have been read)
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
  // (one CTA per row: the list of holes also over the keys, where the movers find it)
  const bool local = SMEM_KEYS && cs == 1;
  for (int i0 = wb; i0 < min(we, a.keep); i0 += 32) {
    const uint32_t kept = kept_bits[(i0 - b) >> 5];
    const uint32_t hole = ~kept & __ballot_sync(0xffffffffu, i0 + lane < min(we, a.keep));
    if ((hole >> lane) & 1u) {
      const uint32_t r = holes + __popc(hole & lt);
      to[r] = i0 + lane;
      if (local) keys[r] = (uint32_t)(i0 + lane);
    }
    holes += __popc(hole);
  }
  cluster_sync();
  // ---- the survivors: weights and positions move here; the rows here or in the second
  // kernel
  const int mb = max(wb, a.keep & ~31);
  for (int i0 = mb; i0 < we; i0 += 32) {
    const uint32_t move = kept_bits[(i0 - b) >> 5] & __ballot_sync(0xffffffffu, i0 + lane >= a.keep);
    if ((move >> lane) & 1u) {
      const uint32_t r = movers + __popc(move & lt);
      const int i = i0 + lane, d = local ? (int)keys[r] : __ldcg(to + r);
      from[r] = i;
      wout[d] = win[i];
      pout[d] = pin[i];
    }
    movers += __popc(move);
  }
  if (a.fused) {
    const int part = ((int)all + cs - 1) / cs;
    cluster_sync();  // the list of survivors is complete
    evict_move<kEvictThreads>(a, m, hk, to, from, min((int)all, (int)rank * part), min((int)all, (int)(rank + 1) * part),
                              reinterpret_cast<long long*>(hist));
  } else if (rank == 0 && tid == 0) {
    a.moves[row] = (int)all;
  }
  cluster_sync();  // the moved weights have been read; no CTA reads another's memory any more
  for (int i = max(b, a.keep) + tid; i < e; i += kEvictThreads) {
    if (!copy_w) wout[i] = 0.0f;
    if (!copy_p) pout[i] = -1;
  }
}

// Segment blockIdx.x of row blockIdx.y's moves.  (An equal share of all moves for each
// of 4 CTAs per SM, though most segments turn out empty here, takes longer: 149 us
// against 133 for both kernels at the size above.  Blocks that are replaced as they
// finish keep more rows under way than blocks that go on from row to row.)
constexpr int kMoveThreads = 256;
__global__ void __launch_bounds__(kMoveThreads, 4) cache_move_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ long long offs[2 * kEvictBatch];
  grid_dep_wait();  // launched while the choosing kernel drains
  const int first = blockIdx.x * a.segment;
  for (int row = blockIdx.y; row < a.M * a.Hkv; row += gridDim.y) {
    const int all = a.moves[row];
    if (first >= all) continue;
    const int* to = a.lists + (size_t)row * 2 * a.list_len;
    evict_move<kMoveThreads>(a, row / a.Hkv, row % a.Hkv, to, to + a.list_len, first, min(all, first + a.segment),
                             offs);
  }
}

// ------------------------------------------------------------------ host side
static long long evict_list_len(long long slots, int keep) {
  const long long rest = slots - keep;
  return rest <= 0 ? 0 : (rest < keep ? rest : keep);
}

size_t evict_workspace_bytes(int M, int Hkv, long long slots, int keep) {
  const long long len = evict_list_len(slots, keep);
  return len == 0 ? 0 : (size_t)M * Hkv * (2 * len + 1) * sizeof(int);
}

template <bool SMEM_KEYS, int THREADS>
static cudaError_t launch_evict_t(const EvictArgs& a, size_t smem, cudaStream_t st) {
  constexpr auto kern = cache_evict_kernel<SMEM_KEYS, THREADS>;
  if (cudaError_t e = allow_smem<kern>(kEvictMaxSmem)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.M * a.Hkv * a.cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

cudaError_t launch_cache_evict(EvictArgs a, void* ws, cudaStream_t st) {
  const int rows = a.M * a.Hkv, sms = sm_count();
  a.list_len = evict_list_len(a.slots, a.keep);
  a.lists = (int*)ws;
  a.moves = a.lists + (size_t)rows * 2 * a.list_len;
  a.fused = a.list_len <= kEvictFused;
  page_divisor(a.page_size, a.page_mul, a.page_shift);
  // Long rows, at most one per SM: 1024 threads each (8191 slots: 12 us to choose from
  // against 20 with 256; 2049 slots: 10.9 against 8.7), and a cluster once its CTAs
  // still have 8192 slots each (14 rows of 32768 slots cut to 4096, in one kernel: 60 us
  // as a CTA each, 44 as two, 34 as four).
  const bool wide = rows <= sms && a.slots >= 4096;
  a.cluster = 1;
  if (wide)
    while (a.cluster < kEvictMaxCluster && 2LL * rows * a.cluster <= sms && a.slots / (2 * a.cluster) >= 8192)
      a.cluster *= 2;
  while (a.cluster < kEvictMaxCluster && a.slots / a.cluster > kEvictMaxSlots / kEvictMaxCluster) a.cluster *= 2;
  const long long share = ((a.slots + a.cluster - 1) / a.cluster + 31) / 32 * 32;
  a.bit_words = (int)((share / 32 + 4) / 4 * 4);
  const size_t fixed = kEvictHistBytes + (size_t)a.bit_words * sizeof(uint32_t);
  cudaError_t e;
  if (share <= kEvictKeys) {
    const size_t smem = fixed + (size_t)share * sizeof(uint32_t);
    e = wide ? launch_evict_t<true, 1024>(a, smem, st) : launch_evict_t<true, 256>(a, smem, st);
  } else {
    e = wide ? launch_evict_t<false, 1024>(a, fixed, st) : launch_evict_t<false, 256>(a, fixed, st);
  }
  if (e != cudaSuccess || a.fused) return e;
  // segments of 256 moves, fewer while that leaves SMs without one
  a.segment = kEvictBatch;
  while (a.segment > 64 && rows * (a.list_len / a.segment) < 4 * sms) a.segment /= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)((a.list_len + a.segment - 1) / a.segment), (unsigned)std::min(rows, 65535));
  return cudaLaunchKernelEx(&cfg, cache_move_kernel, (const EvictArgs)a);
}

}  // namespace aria_q4
