// attn_paged.cu -- attention of one new token per sequence over a paged KV cache.
//
// For sequence m, query head h = hk G + g of key/value head hk, over the n slots
// the sequence holds (its cached ones and, when k_new / v_new are given, the new
// token's own):
//   s_j = scale q[m][h] . k[j][hk]      p_j = exp(s_j - lse), lse = ln sum_j exp(s_j)
//   out[m][h] = sum_j p_j v[j][hk]
// and, for caches that evict, weights[m][hk][j] += sum_g p_j.
//
// The operator reads every K and V row once, 4 bytes per head dimension and slot
// against 4 G flops: it is bound by HBM for every group size that occurs.  So:
//  * one pass with a running maximum and sum per query row; the G query heads of
//    a key/value head share each row that is read;
//  * work is cut along the slots.  The (sequence, head) pairs are laid end to end
//    as tiles of kTile slots and the CTAs take equal contiguous shares of that
//    list, whatever the lengths; a pair that several CTAs share is joined by the
//    last of them to finish (f32 partials in the workspace, added in CTA order,
//    so results do not depend on timing);
//  * each warp streams its own tiles through a cp.async ring in shared memory
//    (16 bytes per lane and copy: any page size and stride works), several tiles
//    ahead and across pair boundaries, so loads never wait for arithmetic;
//  * both products run on warp-level tensor-core MMAs (m16n8k16): rows of A are
//    the query heads.  With at most 8 of them per MMA the other 8 rows carry, in
//    P V, the part of P that rounding to 16 bits drops (p = hi + lo), so the
//    weights of V are exact to ~2^-17 (f16 to 2^-22) at no cost.  tcgen05 has
//    nothing to give here: its 128-row tiles would be 1/128 used at G = 1.
#include <cuda_bf16.h>

#include "q4_common.cuh"
#include "q4_paged.cuh"

namespace aria_q4 {

constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = kPagedWarps * 32;

template <int DH, int RB>
struct PagedCfg {
  static constexpr int kTile = DH <= 32 ? 32 : 16;  // slots per warp and ring stage
  static constexpr int kStageBytes = 2 * kTile * DH * 2;
  static constexpr int kRows = 8 * RB;                              // query heads per pair
  static constexpr int kRedBytes = kPagedWarps * kRows * (DH + 2) * 4;  // the warps' states at a join
  // two CTAs per SM: 113 KB each
  static constexpr int kStagesFit = (110 * 1024 - kRedBytes) / (kPagedWarps * kStageBytes);
  static constexpr int kStages = kStagesFit > 6 ? 6 : kStagesFit < 2 ? 2 : kStagesFit;
  static constexpr int kRingBytes = kPagedWarps * kStages * kStageBytes;
  static constexpr int kMaskBytes = kPagedWarps * kStages * 4;
  static constexpr int kFixedBytes = kRingBytes + kRedBytes + kMaskBytes;
  static constexpr int kPartFloats = kRows * (DH + 2);  // one partial state: O rows, m, l
};

template <bool BF16>
__device__ __forceinline__ void paged_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma_16816(d, a0, a1, a2, a3, b0, b1);
}

// (x, y) rounded to the 16-bit type, and the pair of what the rounding dropped
template <bool BF16>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes, or zeros when !valid (the source is then not read)
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float paged_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// byte offset of the 16-byte chunk c of row r inside a tile: rows of DH * 2
// bytes, chunks permuted so that the 8 rows of an ldmatrix hit 8 bank groups
template <int DH>
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  const int sw = DH == 32 ? (c ^ ((r >> 1) & 3)) : (c ^ (r & 7));
  return (uint32_t)(r * DH * 2 + sw * 16);
}

// The tile list.  Pair (m, hv) -- hv counts the key/value heads, or their chunks
// of query heads -- has ceil(n_m / kTile) tiles; pairs in (m, hv) order.
struct PagedCursor {
  int m, hv, tile, nt;
};

template <int DH, int RB, bool BF16, bool WEIGHTS>
__global__ void __launch_bounds__(kPagedThreads, 2) attn_paged_kernel(const PagedArgs a) {
  using C = PagedCfg<DH, RB>;
  constexpr int TS = C::kTile, S = C::kStages, ROWS = C::kRows, CPR = DH / 8;
  extern __shared__ __align__(128) uint8_t paged_smem[];
  float* red = reinterpret_cast<float*>(paged_smem + C::kRingBytes);
  uint32_t* masks = reinterpret_cast<uint32_t*>(paged_smem + C::kRingBytes + C::kRedBytes);
  int* cum = reinterpret_cast<int*>(paged_smem + C::kFixedBytes);  // [M + 1] tiles of one head before sequence m
  __shared__ int wsum[kPagedWarps];
  __shared__ int s_maxnt;
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;

  // ---- slots of every sequence -> tiles before each
  if (tid == 0) s_maxnt = 0;
  int base = 0;
  for (int m0 = 0; m0 < a.M; m0 += kPagedThreads) {
    const int m = m0 + tid;
    const int nt = m < a.M ? (paged_slots(a, m) + TS - 1) / TS : 0;
    int x = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();  // wsum of the previous round read; s_maxnt set
    if (lane == 31) wsum[warp] = x;
    atomicMax(&s_maxnt, nt);
    __syncthreads();
    int before = base, total = 0;
#pragma unroll
    for (int w = 0; w < kPagedWarps; w++) {
      before += w < warp ? wsum[w] : 0;
      total += wsum[w];
    }
    if (m < a.M) cum[m + 1] = before + x;
    base += total;
  }
  if (tid == 0) cum[0] = 0;
  __syncthreads();
  const long long total = (long long)cum[a.M] * a.Hv;

  // sequences without slots: zeros and an empty log-sum-exp
  for (int m = blockIdx.x; m < a.M; m += gridDim.x) {
    if (cum[m + 1] != cum[m]) continue;
    for (int i = tid; i < a.Hq * DH; i += kPagedThreads)
      reinterpret_cast<uint16_t*>(a.out)[m * a.out_row + (i / DH) * a.out_head + i % DH] = 0;
    for (int h = tid; h < a.Hq; h += kPagedThreads) {
      if (a.lse) a.lse[(size_t)m * a.Hq + h] = -INFINITY;
      if (WEIGHTS) a.lse2[(size_t)m * a.Hq + h] = -INFINITY;
    }
  }
  if (total == 0) return;

  // ---- this CTA's share [t0, t1).  Few short pairs: one whole pair each, which
  // needs no join; else equal shares of at least kMinShare tiles.
  const long long pairs = (long long)a.M * a.Hv;
  const bool whole = pairs <= gridDim.x && s_maxnt <= kPagedWholeTiles;
  const long long want = (total + kPagedMinShare - 1) / kPagedMinShare;
  const long long ctas = whole ? pairs : (want < gridDim.x ? want : (long long)gridDim.x);
  const long long c = blockIdx.x;
  if (c >= ctas) return;
  long long t0, t1;
  PagedCursor seg;
  if (whole) {
    seg.m = (int)(c / a.Hv);
    seg.hv = (int)(c % a.Hv);
    seg.nt = cum[seg.m + 1] - cum[seg.m];
    seg.tile = 0;
    t0 = (long long)cum[seg.m] * a.Hv + (long long)seg.hv * seg.nt;
    t1 = t0 + seg.nt;
  } else {
    t0 = total * c / ctas;
    t1 = total * (c + 1) / ctas;
    int lo = 0, hi = a.M - 1;  // the last m with cum[m] * Hv <= t0 and a tile of its own
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)cum[mid] * a.Hv <= t0) lo = mid; else hi = mid - 1;
    }
    seg.m = lo;
    seg.nt = cum[lo + 1] - cum[lo];
    const long long r = t0 - (long long)cum[lo] * a.Hv;
    seg.hv = seg.nt > 0 ? (int)(r / seg.nt) : 0;
    seg.tile = seg.nt > 0 ? (int)(r - (long long)seg.hv * seg.nt) : 0;
  }
  if (t0 >= t1) return;

  auto next_pair = [&](PagedCursor& p) {  // first tile of the following pair (m = M: none)
    p.tile = 0;
    if (++p.hv < a.Hv) return;
    p.hv = 0;
    do {
      p.m++;
    } while (p.m < a.M && cum[p.m + 1] == cum[p.m]);
    p.nt = p.m < a.M ? cum[p.m + 1] - cum[p.m] : 1;
  };
  auto advance = [&](PagedCursor& p, int step) {
    p.tile += step;
    while (p.m < a.M && p.tile >= p.nt) {
      const int rest = p.tile - p.nt;
      next_pair(p);
      p.tile = rest;
    }
  };

  // ---- producer side of this warp's ring
  uint8_t* ring = paged_smem + warp * (S * C::kStageBytes);
  const uint32_t ring_s = tc_smem_u32(ring);
  uint32_t* mask = masks + warp * S;
  PagedCursor pf = seg;      // next tile to load
  long long pf_t = t0 + warp;
  advance(pf, warp);
  int pf_page = -1;          // page of this lane's row of that tile
  int pf_slots = 0;          // slots of its sequence
  auto lookup = [&]() {
    pf_page = -1;
    if (pf_t >= t1) return;
    pf_slots = paged_slots(a, pf.m);
    const int slot = pf.tile * TS + lane;
    if (lane < TS && slot < pf_slots) {
      const bool is_new = a.k_new != nullptr && slot == pf_slots - 1;
      pf_page = is_new ? -2 : a.table[(long long)pf.m * a.table_stride + slot / a.page_size];
    }
  };
  auto issue = [&](int st) {
    if (pf_t < t1) {
      const int hk = pf.hv / a.chunks;
      const int slot = pf.tile * TS + lane;
      long long off = -1;  // element offset of this lane's row in the pages
      if (pf_page >= 0 && pf_page < a.num_pages)
        off = (long long)pf_page * a.page_stride + (long long)(slot % a.page_size) * a.slot_stride +
              (long long)hk * a.head_stride;
      else if (pf_page == -2)
        off = -2;
      const uint32_t valid = __ballot_sync(0xffffffffu, off != -1);
      if (lane == 0) mask[st] = valid;
      const long long noff = (long long)pf.m * a.new_row + (long long)hk * a.new_head;
      const uint32_t dst = ring_s + st * C::kStageBytes;
#pragma unroll
      for (int i = 0; i < TS * CPR / 32; i++) {
        const int idx = lane + 32 * i, r = idx / CPR, ch = idx % CPR;
        const long long o = __shfl_sync(0xffffffffu, off, r);
        const uint16_t* kp = a.k_pages;
        const uint16_t* vp = a.v_pages;
        if (o >= 0) {
          kp += o + ch * 8;
          vp += o + ch * 8;
        } else if (o == -2) {
          kp = a.k_new + noff + ch * 8;
          vp = a.v_new + noff + ch * 8;
        }
        cp_async_16(dst + tile_off<DH>(r, ch), kp, o != -1);
        cp_async_16(dst + TS * DH * 2 + tile_off<DH>(r, ch), vp, o != -1);
      }
      pf_t += kPagedWarps;
      advance(pf, kPagedWarps);
    }
    cp_async_commit();
    lookup();
  };
  lookup();
#pragma unroll
  for (int s = 0; s < S - 1; s++) issue(s);
  int st = 0;

  // ---- consume: pair by pair
  for (long long t = t0; t < t1;) {
    const int cnt = (int)min((long long)(seg.nt - seg.tile), t1 - t);
    const int first_tile = seg.tile;
    const int hk = seg.hv / a.chunks, h0 = hk * a.G + (seg.hv % a.chunks) * ROWS;  // first query head
    const int rows = min(ROWS, hk * a.G + a.G - h0);
    const int n = paged_slots(a, seg.m);

    // Q fragments: row g (and g + 8) of the A operand, zeros past the pair's heads
    uint32_t qf[DH / 16][2 * RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      const int h = g + 8 * rb;
      const uint16_t* qp = a.q + (long long)seg.m * a.q_row + (long long)(h0 + h) * a.q_head + 2 * t4;
#pragma unroll
      for (int kk = 0; kk < DH / 16; kk++) {
        qf[kk][rb] = h < rows ? *reinterpret_cast<const uint32_t*>(qp + kk * 16) : 0u;
        qf[kk][RB + rb] = h < rows ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8) : 0u;
      }
    }
    float o[RB][DH / 8][4];
    float mx[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      mx[rb] = -INFINITY;
      l[rb] = 0.0f;
#pragma unroll
      for (int j = 0; j < DH / 8; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[rb][j][e] = 0.0f;
    }

    const int skew = (int)((t - t0) % kPagedWarps);
    for (int i = (warp - skew + kPagedWarps) % kPagedWarps; i < cnt; i += kPagedWarps) {
      issue(st == 0 ? S - 1 : st - 1);
      cp_async_wait<S - 1>();
      __syncwarp();
      const uint32_t kt = ring_s + st * C::kStageBytes, vt = kt + TS * DH * 2;
      const uint32_t valid = mask[st];
      const int slot0 = (first_tile + i) * TS;

      // the new token's row goes to the cache from here, once
      if (a.k_new != nullptr && seg.hv % a.chunks == 0 && n - 1 - slot0 < TS && n - 1 >= slot0) {
        const int r = n - 1 - slot0;
        const int page = a.table[(long long)seg.m * a.table_stride + (n - 1) / a.page_size];
        if (page >= 0 && page < a.num_pages && lane < CPR) {
          const long long off = (long long)page * a.page_stride +
                                (long long)((n - 1) % a.page_size) * a.slot_stride + (long long)hk * a.head_stride;
          const uint8_t* sk = ring + st * C::kStageBytes + tile_off<DH>(r, lane);
          *reinterpret_cast<uint4*>(a.k_pages_w + off + lane * 8) = *reinterpret_cast<const uint4*>(sk);
          *reinterpret_cast<uint4*>(a.v_pages_w + off + lane * 8) =
              *reinterpret_cast<const uint4*>(sk + TS * DH * 2);
        }
      }

      // S = Q K^T: columns are slots
      float s[TS / 8][4];
#pragma unroll
      for (int j = 0; j < TS / 8; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[j][e] = 0.0f;
      const int mi = lane >> 3, r8 = lane & 7;
#pragma unroll
      for (int j = 0; j < TS / 16; j++)
#pragma unroll
        for (int kk = 0; kk < DH / 16; kk++) {
          uint32_t b[4];
          ldsm_x4(kt + tile_off<DH>(16 * j + (mi >> 1) * 8 + r8, 2 * kk + (mi & 1)), b);
          const uint32_t a1 = RB == 2 ? qf[kk][1] : 0u, a3 = RB == 2 ? qf[kk][2 * RB - 1] : 0u;
          paged_mma<BF16>(s[2 * j], qf[kk][0], a1, qf[kk][RB], a3, b[0], b[1]);
          paged_mma<BF16>(s[2 * j + 1], qf[kk][0], a1, qf[kk][RB], a3, b[2], b[3]);
        }

      // scores to the log2 domain; slots past the end or without a page are -inf
      uint32_t ph[RB][TS / 8], pl[RB][TS / 8];
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        float m_new = mx[rb];
#pragma unroll
        for (int j = 0; j < TS / 8; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float& x = s[j][2 * rb + e];
            x = (valid >> (8 * j + 2 * t4 + e)) & 1u ? x * a.scale_log2 : -INFINITY;
            m_new = fmaxf(m_new, x);
          }
        if (WEIGHTS) {
          const int h = g + 8 * rb;
          float* sp = a.scores + ((size_t)seg.m * a.Hq + h0 + h) * a.score_row + slot0 + 2 * t4;
#pragma unroll
          for (int j = 0; j < TS / 8; j++)
            if (h < rows && slot0 + 8 * j + 2 * t4 < n)  // the row's stride is even: both fit
              *reinterpret_cast<float2*>(sp + 8 * j) = make_float2(s[j][2 * rb], s[j][2 * rb + 1]);
        }
        m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 1));
        m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 2));
        // a row that has seen no slot yet keeps -inf; its p are then 0, not NaN
        const float msub = m_new == -INFINITY ? 0.0f : m_new;
        if (__any_sync(0xffffffffu, m_new > mx[rb])) {
          const float alpha = paged_ex2(mx[rb] - msub);
          l[rb] *= alpha;
#pragma unroll
          for (int j = 0; j < DH / 8; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[rb][j][e] *= alpha;
          mx[rb] = m_new;
        }
#pragma unroll
        for (int j = 0; j < TS / 8; j++) {
          const float p0 = paged_ex2(s[j][2 * rb] - msub), p1 = paged_ex2(s[j][2 * rb + 1] - msub);
          l[rb] += p0 + p1;
          split_pair<BF16>(p0, p1, ph[rb][j], pl[rb][j]);
        }
      }

      // O += P V: rows 0-7 the rounded weights, rows 8-15 what the rounding dropped
#pragma unroll
      for (int j = 0; j < TS / 16; j++)
#pragma unroll
        for (int d = 0; d < DH / 16; d++) {
          uint32_t b[4];
          ldsm_x4_trans(vt + tile_off<DH>(16 * j + (mi & 1) * 8 + r8, 2 * d + (mi >> 1)), b);
#pragma unroll
          for (int rb = 0; rb < RB; rb++) {
            paged_mma<BF16>(o[rb][2 * d], ph[rb][2 * j], pl[rb][2 * j], ph[rb][2 * j + 1], pl[rb][2 * j + 1], b[0],
                            b[1]);
            paged_mma<BF16>(o[rb][2 * d + 1], ph[rb][2 * j], pl[rb][2 * j], ph[rb][2 * j + 1], pl[rb][2 * j + 1],
                            b[2], b[3]);
          }
        }
      __syncwarp();  // the stage may be refilled
      st = st + 1 == S ? 0 : st + 1;
    }

    // ---- the warps' states of this pair -> shared memory -> one state
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 1);
      l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 2);
      const int h = g + 8 * rb;
      float* ro = red + (warp * ROWS + h) * DH;
      if (h < rows) {
#pragma unroll
        for (int j = 0; j < DH / 8; j++)
          *reinterpret_cast<float2*>(ro + 8 * j + 2 * t4) =
              make_float2(o[rb][j][0] + o[rb][j][2], o[rb][j][1] + o[rb][j][3]);
        if (t4 == 0) {
          red[kPagedWarps * ROWS * DH + warp * ROWS + h] = mx[rb];
          red[kPagedWarps * ROWS * (DH + 1) + warp * ROWS + h] = l[rb];
        }
      }
    }
    __syncthreads();
    const float* rm = red + kPagedWarps * ROWS * DH;
    const float* rl = rm + kPagedWarps * ROWS;
    const bool alone = cnt == seg.nt;
    const long long f = (long long)cum[seg.m] * a.Hv + (long long)seg.hv * seg.nt;  // the pair's first tile
    float* part = a.parts + (size_t)(2 * c + (f <= t0 ? 0 : 1)) * C::kPartFloats;
    for (int i = tid; i < rows * DH; i += kPagedThreads) {
      const int h = i / DH, d = i % DH;
      float m = rm[h];
#pragma unroll
      for (int w = 1; w < kPagedWarps; w++) m = fmaxf(m, rm[w * ROWS + h]);
      const float ms = m == -INFINITY ? 0.0f : m;
      float acc = 0.0f, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kPagedWarps; w++) {
        const float e = paged_ex2(rm[w * ROWS + h] - ms);
        acc = fmaf(e, red[(w * ROWS + h) * DH + d], acc);
        sum = fmaf(e, rl[w * ROWS + h], sum);
      }
      if (alone) {
        paged_store<BF16>(a, seg.m, h0 + h, d, sum > 0.0f ? acc / sum : 0.0f);
        if (d == 0) paged_store_lse<WEIGHTS>(a, seg.m, h0 + h, m, sum);
      } else {
        part[i] = acc;
        if (d == 0) {
          part[ROWS * DH + h] = m;
          part[ROWS * DH + ROWS + h] = sum;
        }
      }
    }
    if (!alone) {
      // the last CTA of the pair to arrive adds the partial states in CTA order
      const long long last_t = f + seg.nt - 1;
      const int c0 = (int)(((f + 1) * ctas - 1) / total), c1 = (int)(((last_t + 1) * ctas - 1) / total);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        unsigned* cnt_p = a.counters + c0;  // a CTA begins at most one pair that it does not finish
        const unsigned prev = atomicAdd(cnt_p, 1u);
        s_last = prev == (unsigned)(c1 - c0);
        if (s_last) *cnt_p = 0;  // ready for the next call
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int i = tid; i < rows * DH; i += kPagedThreads) {
          const int h = i / DH, d = i % DH;
          float m = -INFINITY, acc = 0.0f, sum = 0.0f;
          for (int k = c0; k <= c1; k++) {
            const long long kt0 = total * k / ctas;
            const float* p = a.parts + (size_t)(2 * k + (f <= kt0 ? 0 : 1)) * C::kPartFloats;
            const float pm = __ldcg(p + ROWS * DH + h), ps = __ldcg(p + ROWS * DH + ROWS + h), po = __ldcg(p + i);
            const float m2 = fmaxf(m, pm), ms = m2 == -INFINITY ? 0.0f : m2;
            const float e0 = paged_ex2(m - ms), e1 = paged_ex2(pm - ms);
            acc = fmaf(acc, e0, po * e1);
            sum = fmaf(sum, e0, ps * e1);
            m = m2;
          }
          paged_store<BF16>(a, seg.m, h0 + h, d, sum > 0.0f ? acc / sum : 0.0f);
          if (d == 0) paged_store_lse<WEIGHTS>(a, seg.m, h0 + h, m, sum);
        }
      }
    }
    __syncthreads();  // red may be written again
    t += cnt;
    next_pair(seg);
  }
  cp_async_wait<0>();
}

// weights_out[m][hk][j] = weights_in[m][hk][j] (0 for the new token's slot) +
// sum over the group's heads of 2^(score - lse2), the scores as the attention
// kernel left them; slot_pos of the new token's slot.  Slots past the end are
// not touched.  4 G + 8 bytes per slot, from L2 mostly: bound by its launch.
__global__ void __launch_bounds__(256) paged_weights_kernel(const PagedArgs a, const float* win, float* wout,
                                                            long long cap, int* slot_pos, const int* positions) {
  const int m = blockIdx.z, hk = blockIdx.y;
  const int n = paged_slots(a, m);
  const int old = n > 0 && a.k_new != nullptr ? n - 1 : n;
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  const size_t at = ((size_t)m * a.Hkv + hk) * cap + j;
  float w = j < old ? win[at] : 0.0f;
  for (int g = 0; g < a.G; g++) {
    const size_t h = (size_t)m * a.Hq + hk * a.G + g;
    const float ls = a.lse2[h];
    if (ls != -INFINITY) w += paged_ex2(a.scores[h * a.score_row + j] - ls);
  }
  wout[at] = w;
  if (j >= old && slot_pos) slot_pos[at] = positions[m];
}

// ------------------------------------------------------------------ host side
static int paged_chunks(int DH, int G) {
  const int rows = G <= 8 || DH == 256 ? 8 : 16;
  return (G + rows - 1) / rows;
}

static int paged_grid() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return 2 * sms;
}

static size_t paged_part_bytes(int DH, int G) {
  const int rows = G <= 8 || DH == 256 ? 8 : 16;
  return align_up((size_t)2 * paged_grid() * rows * (DH + 2) * sizeof(float), 256);
}

// Workspace: one counter per CTA (zero between calls; a region of fixed size, so
// that calls of any shape may follow one another), partial states, and for the
// accumulated weights one log-sum-exp and score_row scores per query head.
static size_t paged_counter_bytes() { return align_up((size_t)paged_grid() * sizeof(unsigned), 256); }

size_t paged_workspace_bytes(int M, int Hq, int Hkv, int DH, long long slots, bool weights) {
  const int G = Hq / Hkv;
  size_t b = paged_counter_bytes() + paged_part_bytes(DH, G);
  if (weights) b += align_up((size_t)M * Hq * sizeof(float), 256) + (size_t)M * Hq * align_up(slots, 4) * sizeof(float);
  return b;
}

template <int DH, int RB, bool BF16, bool WEIGHTS>
static cudaError_t launch_paged_t(const PagedArgs& a, cudaStream_t st) {
  using C = PagedCfg<DH, RB>;
  const size_t smem = C::kFixedBytes + (size_t)(a.M + 1) * sizeof(int);
  auto kern = attn_paged_kernel<DH, RB, BF16, WEIGHTS>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kern<<<paged_grid(), kPagedThreads, smem, st>>>(a);
  return cudaGetLastError();
}

template <int DH, int RB>
static cudaError_t launch_paged_d(const PagedArgs& a, bool bf16, bool weights, cudaStream_t st) {
  if (bf16)
    return weights ? launch_paged_t<DH, RB, true, true>(a, st) : launch_paged_t<DH, RB, true, false>(a, st);
  return weights ? launch_paged_t<DH, RB, false, true>(a, st) : launch_paged_t<DH, RB, false, false>(a, st);
}

cudaError_t launch_attention_paged(PagedArgs a, int DH, bool bf16, void* ws, const float* win, float* wout,
                                   long long cap, int* slot_pos, const int* positions, cudaStream_t st) {
  const bool weights = wout != nullptr;
  a.chunks = paged_chunks(DH, a.G);
  a.Hv = a.Hkv * a.chunks;
  uint8_t* w = (uint8_t*)ws;
  a.counters = (unsigned*)w;
  w += paged_counter_bytes();
  a.parts = (float*)w;
  w += paged_part_bytes(DH, a.G);
  a.score_row = (long long)align_up((size_t)a.slots, 4);
  if (weights) {
    a.lse2 = (float*)w;
    w += align_up((size_t)a.M * a.Hq * sizeof(float), 256);
    a.scores = (float*)w;
  }
  cudaError_t e = cudaErrorInvalidValue;
  const bool two = a.G > 8;
  switch (DH) {
    case 32: e = two ? launch_paged_d<32, 2>(a, bf16, weights, st) : launch_paged_d<32, 1>(a, bf16, weights, st); break;
    case 64: e = two ? launch_paged_d<64, 2>(a, bf16, weights, st) : launch_paged_d<64, 1>(a, bf16, weights, st); break;
    case 128:
      e = two ? launch_paged_d<128, 2>(a, bf16, weights, st) : launch_paged_d<128, 1>(a, bf16, weights, st);
      break;
    case 256: e = launch_paged_d<256, 1>(a, bf16, weights, st); break;
  }
  if (e != cudaSuccess || !weights) return e;
  paged_weights_kernel<<<dim3((unsigned)((a.slots + 255) / 256), a.Hkv, a.M), 256, 0, st>>>(a, win, wout, cap,
                                                                                        slot_pos, positions);
  return cudaGetLastError();
}

}  // namespace aria_q4
