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
//    as tiles of kTile slots, and the grid's warps take equal contiguous parts of
//    that list, whatever the lengths.  A pair within one warp's part is finished in
//    its registers; the others leave f32 partial states in the workspace (a CTA that
//    is inside one pair joins its four warps' first), and the last to arrive adds a
//    pair's states in list order, so results do not depend on timing;
//  * each warp streams its own tiles through a cp.async ring in shared memory,
//    several tiles ahead and across pair boundaries, so loads never wait for
//    arithmetic;
//  * a maximum passes NaN over, a sum does not: a row's sum is 0 exactly when nothing
//    was there to attend over, and NaN when a score was NaN or +inf.  So the sum
//    alone says whether a state is empty, and NaN reaches out, lse and the weights
//    whichever way a pair is cut;
//  * both products run on warp-level tensor-core MMAs (m16n8k16): rows of A are
//    the query heads.  With at most 8 of them per MMA the other 8 rows carry, in
//    P V, the part of P that rounding to 16 bits drops (p = hi + lo).  bf16 holds
//    the weights of V to 2^-17 of themselves; f16, whose smallest step is 2^-24,
//    holds 2^15 p, so the weights are right to 2^-22 of themselves or 2^-40 of the
//    largest, whichever is more (unscaled, a slot 17 behind the leading one was
//    lost, and with it all of 32749 such slots).  tcgen05 has nothing to give here:
//    its 128-row tiles would be 1/128 used at G = 1.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "q4_common.cuh"
#include "q4_paged.cuh"
#include "q4_status.cuh"

namespace aria_q4 {

constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = kPagedWarps * 32;

template <int DH, int RB>
struct PagedCfg {
  static constexpr int kTile = DH <= 64 ? 32 : 16;  // slots per ring stage
  static constexpr int kRows = 8 * RB;              // query heads per pair
  static constexpr int kKBytes = kTile * DH * 2;
  static constexpr int kStageBytes = 2 * kKBytes;   // K, V
};
constexpr int kPagedMaxStages = 6;

// Floats of a state of `rows` query heads: O rows, then their maxima, then their
// sums; a multiple of 4 for 16-byte loads.
__host__ __device__ constexpr int paged_state_floats(int dh, int rows) { return (rows * (dh + 2) + 3) / 4 * 4; }

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

// What p (at most 1) is multiplied by for the product with V, and its inverse: powers
// of two, so both are exact.
template <bool BF16>
struct PagedP {
  static constexpr float kUp = BF16 ? 1.0f : 32768.0f, kDown = 1.0f / kUp;
};

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
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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

// The tile list cut into parts, one per warp: the first `more` of size + 1 tiles.
struct PagedCut {
  int size, more;
  __device__ PagedCut(int total, int parts) : size(total / parts), more(total % parts) {}
  __device__ int begin(int part) const { return part * size + min(part, more); }
  __device__ int part_of(int t) const {
    const int longer = more * (size + 1);
    return t < longer ? t / (size + 1) : more + (t - longer) / size;
  }
};

// One warp: the partial states of the pair at tiles [f, f + nt) of the list -> rows
// h_first, h_first + h_step, ... of its output.  offs: shared memory for an int per part
// that the pair touches.  The loads of a row's first 16 states go out together with
// those of their maxima and sums: one round trip where a pair has no more.
template <int DH, int ROWS, bool BF16, bool WEIGHTS>
__device__ __noinline__ void paged_join(const PagedArgs& a, const PagedCut cut, int f, int nt, int m, int h0,
                                        int rows, int* offs, int h_first, int h_step) {
  constexpr int VEC = DH >= 128 ? 4 : DH / 32;  // floats per lane and load
  constexpr int UN = 16;                        // states per batch of loads
  const int lane = threadIdx.x & 31, srows = min(a.G, ROWS), sf = paged_state_floats(DH, srows);
  // the parts' states, in order: a CTA inside the pair has one for all four
  const int p0 = cut.part_of(f), p1 = cut.part_of(f + nt - 1);
  int cnt = 0;
  for (int pb = p0; pb <= p1; pb += 32) {
    const int part = pb + lane, c = part / kPagedWarps * kPagedWarps;
    const bool inside = cut.begin(c) >= f && cut.begin(c + kPagedWarps) <= f + nt;
    const bool on = part <= p1 && (!inside || part == c);
    const unsigned all = __ballot_sync(0xffffffffu, on);
    if (on) offs[cnt + __popc(all & ((1u << lane) - 1u))] = (2 * part + (f <= cut.begin(part) ? 0 : 1)) * sf;
    cnt += __popc(all);
  }
  __syncwarp();
#pragma unroll 1
  for (int h = h_first; h < rows; h += h_step) {
#pragma unroll 1
    for (int d0 = lane * VEC; d0 < DH; d0 += 32 * VEC) {
      const float* col = a.parts + h * DH + d0;
      const float* stat = a.parts + srows * DH + h;
      float x[UN][VEC];
      auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < UN; u++) {
          const float* p = col + offs[min(base + u, cnt - 1)];
          if (VEC == 4)
            *reinterpret_cast<float4*>(x[u]) = __ldcg(reinterpret_cast<const float4*>(p));
          else if (VEC == 2)
            *reinterpret_cast<float2*>(x[u]) = __ldcg(reinterpret_cast<const float2*>(p));
          else
            x[u][0] = __ldcg(p);
        }
      };
      load(0);
      // every lane's states -> one maximum, the sum of their sums against it
      float mx = -INFINITY, l = 0.0f;
      for (int k = lane; k < cnt; k += 32) {
        const float km = __ldcg(stat + offs[k]), kl = __ldcg(stat + offs[k] + srows), m2 = fmaxf(mx, km);
        const float ms = m2 == -INFINITY ? 0.0f : m2;
        l = l * paged_ex2(mx - ms) + kl * paged_ex2(km - ms);
        mx = m2;
      }
      float top = mx;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float ms = top == -INFINITY ? 0.0f : top;
      l *= paged_ex2(mx - ms);
      float w = cnt <= 32 ? paged_ex2(mx - ms) : 0.0f;  // up to 32 states: lane k's maximum is state k's
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      float acc[VEC];
#pragma unroll
      for (int v = 0; v < VEC; v++) acc[v] = 0.0f;
#pragma unroll 1
      for (int base = 0; base < cnt; base += UN) {
        if (base > 0) load(base);
        if (cnt > 32 && base % 32 == 0)
          w = base + lane < cnt ? paged_ex2(__ldcg(stat + offs[base + lane]) - ms) : 0.0f;
#pragma unroll
        for (int u = 0; u < UN; u++) {
          const float wu = __shfl_sync(0xffffffffu, w, base % 32 + u);  // 0 past the last
#pragma unroll
          for (int v = 0; v < VEC; v++) acc[v] = fmaf(wu, x[u][v], acc[v]);
        }
      }
#pragma unroll
      for (int v = 0; v < VEC; v++) paged_store<BF16>(a, m, h0 + h, d0 + v, acc[v] * inv);
      if (d0 == 0) paged_store_lse<WEIGHTS>(a, m, h0 + h, top, l);
    }
  }
}

// PAGE16: pages of a multiple of 16 slots, so that 16 slots of a tile share a page
// and their addresses are one base and a stride; otherwise every row has its own.
template <int DH, int RB, bool BF16, bool WEIGHTS, bool PAGE16>
__global__ void __launch_bounds__(kPagedThreads, 2) attn_paged_kernel(const __grid_constant__ PagedArgs a) {
  using C = PagedCfg<DH, RB>;
  constexpr int TS = C::kTile, ROWS = C::kRows, CPR = DH / 8;
  constexpr int RPI = 32 / (CPR < 32 ? CPR : 32);  // rows per warp-wide copy
  extern __shared__ __align__(128) uint8_t paged_smem[];
  const int S = a.stages;                                 // of every warp's ring
  const int srows = min(a.G, ROWS);                       // rows of a state
  const int sf = paged_state_floats(DH, srows);
  int* cum = reinterpret_cast<int*>(paged_smem + kPagedWarps * S * C::kStageBytes);  // [M + 1] tiles before m
  int* slots = cum + a.M + 1;                                                       // [M]
  __shared__ int wsum[kPagedWarps];
  __shared__ int s_maxnt, s_last;
  __shared__ uint32_t masks[kPagedWarps][kPagedMaxStages];  // per ring stage: the slots that are there
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3, r8 = lane & 7;

  // ---- slots of every sequence -> tiles before each
  if (tid == 0) {
    s_maxnt = 0;
    cum[0] = 0;
  }
  if (WEIGHTS) grid_dep_launch();
  int base = 0;
  for (int m0 = 0; m0 < a.M; m0 += kPagedThreads) {
    const int m = m0 + tid;
    const int n = m < a.M ? paged_slots(a, m) : 0;
    const int nt = (n + TS - 1) / TS;
    int x = nt, mx = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    __syncthreads();  // wsum of the previous round read; s_maxnt set
    if (lane == 31) {
      wsum[warp] = x;
      atomicMax(&s_maxnt, mx);
    }
    __syncthreads();
    int before = base;
#pragma unroll
    for (int w = 0; w < kPagedWarps; w++) {
      before += w < warp ? wsum[w] : 0;
      base += wsum[w];
    }
    if (m < a.M) {
      cum[m + 1] = before + x;
      slots[m] = n;
    }
  }
  __syncthreads();
  const int total = cum[a.M] * a.Hv;

  // sequences without slots: zeros and an empty log-sum-exp
  for (int m = blockIdx.x; m < a.M; m += gridDim.x) {
    if (slots[m] != 0) continue;
    for (int i = tid; i < a.Hq * DH; i += kPagedThreads)
      a.out[m * a.out_row + (i / DH) * a.out_head + i % DH] = 0;
    for (int h = tid; h < a.Hq; h += kPagedThreads) {
      if (a.lse) a.lse[(size_t)m * a.Hq + h] = -INFINITY;
      if (WEIGHTS) a.lse2[(size_t)m * a.Hq + h] = -INFINITY;
    }
  }
  if (total == 0) return;

  // ---- this CTA's share [t0, t1).  Few short pairs: one whole pair each, which
  // needs no join across CTAs; else equal shares of at least kPagedMinSlots.
  const int pairs = a.M * a.Hv;
  const bool whole = pairs <= (int)gridDim.x && s_maxnt * TS <= kPagedWholeSlots;
  const int ctas = whole ? pairs : min(max(1, total / (kPagedMinSlots / TS)), (int)gridDim.x);
  const int c = blockIdx.x;
  if (c >= ctas) return;
  const PagedCut cut(total, ctas * kPagedWarps);
  int t0, t1, w0, w1;
  if (whole) {
    const int m = c / a.Hv, nt = cum[m + 1] - cum[m];
    t0 = cum[m] * a.Hv + (c % a.Hv) * nt;
    t1 = t0 + nt;
    w0 = t0 + nt * warp / kPagedWarps;
    w1 = t0 + nt * (warp + 1) / kPagedWarps;
  } else {
    t0 = cut.begin(c * kPagedWarps);
    t1 = cut.begin(c * kPagedWarps + kPagedWarps);
    w0 = cut.begin(c * kPagedWarps + warp);
    w1 = cut.begin(c * kPagedWarps + warp + 1);
  }
  if (t0 >= t1) return;

  // the pair and tile at position t of the list
  auto locate = [&](int t) {
    PagedCursor p;
    int lo = 0, hi = a.M - 1;  // the last m with cum[m] Hv <= t: empty sequences before it share its start
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] * a.Hv <= t) lo = mid; else hi = mid - 1;
    }
    p.m = lo;
    p.nt = cum[lo + 1] - cum[lo];
    const int r = t - cum[lo] * a.Hv;
    p.hv = r / p.nt;
    p.tile = r - p.hv * p.nt;
    return p;
  };
  auto next_pair = [&](PagedCursor& p) {  // to the following pair's first tile
    p.tile = 0;
    if (++p.hv < a.Hv) return;
    p.hv = 0;
    do {
      p.m++;
    } while (p.m < a.M && slots[p.m] == 0);
    p.nt = p.m < a.M ? cum[p.m + 1] - cum[p.m] : 1;
  };

  uint8_t* ring = paged_smem + warp * (S * C::kStageBytes);
  const uint32_t ring_s = tc_smem_u32(ring);
  // a share that lies within one pair: the warps' states are joined here
  const PagedCursor pair0 = locate(t0);
  const int pair0_t = t0 - pair0.tile;
  const bool inside = t1 <= pair0_t + pair0.nt;
  if (inside && w0 >= w1 && lane < srows) {  // (a warp without a tile has an empty state)
    reinterpret_cast<float*>(ring)[srows * DH + lane] = -INFINITY;
    reinterpret_cast<float*>(ring)[srows * DH + srows + lane] = 0.0f;
  }

  if (w0 < w1) {
    PagedCursor seg = locate(w0);
    PagedCursor open[2] = {seg, seg};  // pairs that reach past this warp's part: at its start, at its end
    int open_t[2] = {-1, -1};          // their first tiles
    int at = w0;                       // position of seg's tile in the list

    // ---- producer side of this warp's ring: pf is the next tile to load
    PagedCursor pf = seg;
    int left = w1 - w0;
    constexpr uint32_t kAll = TS == 32 ? 0xffffffffu : (1u << (TS & 31)) - 1u;
    const int r0 = lane / CPR, ch = lane % CPR;  // this lane's row of a warp-wide copy, and its 16 bytes
    const long long lane_src = r0 * a.slot_stride + ch * 8, copy_step = RPI * a.slot_stride;
    int page = -1;      // of this lane's rows of that tile (PAGE16: lanes 0-15 its first 16 slots, ...)
    auto page_index = [&](int slot) { return (int)(((unsigned long long)(unsigned)slot * a.page_mul) >> a.page_shift); };
    auto lookup = [&]() {
      page = -1;
      if (left <= 0) return;
      const int slot = pf.tile * TS + (PAGE16 ? lane & ~15 : lane);
      if (slot < slots[pf.m] && (PAGE16 ? TS == 32 || lane < 16 : lane < TS)) {
        const int e = a.table[(long long)pf.m * a.table_stride + page_index(slot)];
        page = e < a.num_pages ? e : -1;
      }
    };
    auto issue = [&](int st) {
      if (left > 0) {
        const int hk = a.chunks == 1 ? pf.hv : pf.hv / a.chunks;
        const int slot0 = pf.tile * TS, have = slots[pf.m] - slot0;  // slots of the pair from here on
        const uint32_t dst = ring_s + st * C::kStageBytes;
        int last = a.k_new != nullptr && have <= TS ? have - 1 : TS;  // row of the new token, if here
        const long long noff = (long long)pf.m * a.new_row + (long long)hk * a.new_head;
        uint32_t valid;
        if (PAGE16) {
          constexpr int HALVES = TS / 16;
          long long off[HALVES];
          int rows[HALVES];
          valid = 0;
#pragma unroll
          for (int h = 0; h < HALVES; h++) {
            const int pg = __shfl_sync(0xffffffffu, page, 16 * h);
            const int slot = slot0 + 16 * h;
            off[h] = (long long)pg * a.page_stride + (long long)(slot - page_index(slot) * a.page_size) * a.slot_stride +
                     (long long)hk * a.head_stride;
            rows[h] = pg < 0 ? 0 : min(16, max(0, have - 16 * h));
            valid |= ((1u << rows[h]) - 1u) << (16 * h);
          }
          if (valid == kAll && last == TS) {
            // a whole tile of the pages: one address per half, a constant step per copy
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
              const uint16_t* kp = a.k_pages + off[h] + lane_src;
              const uint16_t* vp = a.v_pages + off[h] + lane_src;
#pragma unroll
              for (int i = 16 / RPI * h; i < 16 / RPI * (h + 1); i++) {
                cp_async_16(dst + tile_off<DH>(RPI * i + r0, ch), kp);
                cp_async_16(dst + C::kKBytes + tile_off<DH>(RPI * i + r0, ch), vp);
                kp += copy_step;
                vp += copy_step;
              }
            }
          } else {
            // (valid has the new token's bit where its page exists; elsewhere its slot is absent
            // like any other)
            if (last < TS && !((valid >> last) & 1u)) last = TS;
#pragma unroll
            for (int i = 0; i < TS * CPR / 32; i++) {
              const int rh = RPI * i;  // first row of this copy; all of one half
              const int r = rh + r0, rr = r - (rh & ~15);
              const bool ok = rr < rows[rh / 16];
              long long o = ok ? off[rh / 16] + (long long)rr * a.slot_stride + ch * 8 : 0;
              const uint16_t* kp = a.k_pages + o;
              const uint16_t* vp = a.v_pages + o;
              if (r == last) {
                kp = a.k_new + noff + ch * 8;
                vp = a.v_new + noff + ch * 8;
              }
              cp_async_16(dst + tile_off<DH>(r, ch), kp, ok || r == last);
              cp_async_16(dst + C::kKBytes + tile_off<DH>(r, ch), vp, ok || r == last);
            }
          }
        } else {
          const int slot = slot0 + lane;
          long long off = -1;  // element offset of this lane's row in the pages
          if (page >= 0 && lane == last)
            off = -2;
          else if (page >= 0)
            off = (long long)page * a.page_stride + (long long)(slot - page_index(slot) * a.page_size) * a.slot_stride +
                  (long long)hk * a.head_stride;
          valid = __ballot_sync(0xffffffffu, off != -1);
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
            cp_async_16(dst + C::kKBytes + tile_off<DH>(r, ch), vp, o != -1);
          }
        }
        if (lane == 0) masks[warp][st] = valid;
        left--;
        if (++pf.tile == pf.nt) next_pair(pf);
      }
      cp_async_commit();
      lookup();
    };
    lookup();
    for (int s = 0; s < S - 1; s++) issue(s);
    int st = 0;

    // ---- consume, pair by pair
    for (int todo = w1 - w0; todo > 0;) {
      const int begin = seg.tile, end = min(seg.nt, begin + todo);
      todo -= end - begin;
      const int hk = a.chunks == 1 ? seg.hv : seg.hv / a.chunks, chunk = seg.hv - hk * a.chunks;
      const int h0 = hk * a.G + chunk * ROWS;  // first query head
      const int rows = min(ROWS, (hk + 1) * a.G - h0);
      const int n = slots[seg.m];
      // A fragments of Q.  Rows past the pair's heads repeat its first one: the rows
      // of the products do not mix, and theirs are not kept.
      uint32_t qf[DH / 16][2 * RB];
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        const int h = g + 8 * rb < rows ? g + 8 * rb : 0;
        const uint16_t* qp = a.q + (long long)seg.m * a.q_row + (long long)(h0 + h) * a.q_head + 2 * t4;
#pragma unroll
        for (int kk = 0; kk < DH / 16; kk++) {
          qf[kk][rb] = *reinterpret_cast<const uint32_t*>(qp + kk * 16);
          qf[kk][RB + rb] = *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8);
        }
      }
      float o[RB][DH / 8][4];
      // maximum and sum; l_off: what rounding has put too much into the sum, taken out of
      // the next tile's (small weights after a large one would otherwise not count)
      float mx[RB], l[RB], l_off[RB];
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        mx[rb] = -INFINITY;
        l[rb] = l_off[rb] = 0.0f;
#pragma unroll
        for (int j = 0; j < DH / 8; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[rb][j][e] = 0.0f;
      }

      for (int tile = begin; tile < end; tile++) {
        issue(st == 0 ? S - 1 : st - 1);
        switch (S) {  // all but the newest S - 1 groups have arrived
          case 2: cp_async_wait<1>(); break;
          case 3: cp_async_wait<2>(); break;
          case 4: cp_async_wait<3>(); break;
          case 5: cp_async_wait<4>(); break;
          default: cp_async_wait<5>(); break;
        }
        __syncwarp();
        const uint32_t kt = ring_s + st * C::kStageBytes, vt = kt + C::kKBytes;
        const uint32_t valid = masks[warp][st];
        const int slot0 = tile * TS;

        // the new token's row goes to the cache from here, once
        if (a.k_new != nullptr && tile == seg.nt - 1 && chunk == 0 && lane < CPR) {
          const int r = n - 1 - slot0, pi = page_index(n - 1);
          const int pg = a.table[(long long)seg.m * a.table_stride + pi];
          if (pg >= 0 && pg < a.num_pages) {
            const long long off = (long long)pg * a.page_stride + (long long)(n - 1 - pi * a.page_size) * a.slot_stride +
                                  (long long)hk * a.head_stride + lane * 8;
            const uint8_t* sk = ring + st * C::kStageBytes + tile_off<DH>(r, lane);
            *reinterpret_cast<uint4*>(a.k_pages_w + off) = *reinterpret_cast<const uint4*>(sk);
            *reinterpret_cast<uint4*>(a.v_pages_w + off) = *reinterpret_cast<const uint4*>(sk + C::kKBytes);
          }
        }

        // S = Q K^T: columns are slots
        float s[TS / 8][4];
#pragma unroll
        for (int j = 0; j < TS / 8; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[j][e] = 0.0f;
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
#pragma unroll
          for (int j = 0; j < TS / 8; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) s[j][2 * rb + e] *= a.scale_log2;
          if (valid != kAll) {
#pragma unroll
            for (int j = 0; j < TS / 8; j++)
#pragma unroll
              for (int e = 0; e < 2; e++)
                if (!((valid >> (8 * j + 2 * t4 + e)) & 1u)) s[j][2 * rb + e] = -INFINITY;
          }
          float m_new = mx[rb];
#pragma unroll
          for (int j = 0; j < TS / 8; j++) m_new = fmaxf(m_new, fmaxf(s[j][2 * rb], s[j][2 * rb + 1]));
          if (WEIGHTS) {
            const int h = g + 8 * rb;
            if (h < rows) {
              float* sp = a.scores + ((size_t)seg.m * a.Hq + h0 + h) * a.score_row + slot0 + 2 * t4;
#pragma unroll
              for (int j = 0; j < TS / 8; j++)
                if (slot0 + 8 * j + 2 * t4 < n)  // the row's stride is even: both fit
                  *reinterpret_cast<float2*>(sp + 8 * j) = make_float2(s[j][2 * rb], s[j][2 * rb + 1]);
            }
          }
          m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 1));
          m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 2));
          // a row that has seen no slot yet keeps -inf; its p are then 0, not NaN
          const float msub = m_new == -INFINITY ? 0.0f : m_new;
          if (__any_sync(0xffffffffu, m_new > mx[rb])) {
            const float alpha = paged_ex2(mx[rb] - msub);
            l[rb] *= alpha;
            l_off[rb] *= alpha;
#pragma unroll
            for (int j = 0; j < DH / 8; j++)
#pragma unroll
              for (int e = 0; e < 4; e++) o[rb][j][e] *= alpha;
            mx[rb] = m_new;
          }
          float sum = -l_off[rb];
#pragma unroll
          for (int j = 0; j < TS / 8; j++) {
            const float p0 = paged_ex2(s[j][2 * rb] - msub), p1 = paged_ex2(s[j][2 * rb + 1] - msub);
            sum += p0 + p1;
            split_pair<BF16>(p0 * PagedP<BF16>::kUp, p1 * PagedP<BF16>::kUp, ph[rb][j], pl[rb][j]);
          }
          const float l_new = l[rb] + sum;
          l_off[rb] = (l_new - l[rb]) - sum;
          l[rb] = l_new;
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

      // ---- this warp's state of the pair: finished, or partial
      const bool all = !inside && begin == 0 && end == seg.nt;
      const int f = at - begin;  // the pair's first tile
      const int side = f <= w0 ? 0 : 1;
      float* state = a.parts + (2 * (c * kPagedWarps + warp) + side) * sf;
      if (inside) {  // the warp's only pair: its ring is free
        cp_async_wait<0>();
        __syncwarp();
        state = reinterpret_cast<float*>(ring);
      }
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 1);
        l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 2);
        const int h = g + 8 * rb;
        if (h >= rows) continue;
        if (all) {
          const float inv = l[rb] == 0.0f ? 0.0f : PagedP<BF16>::kDown / l[rb];
#pragma unroll
          for (int j = 0; j < DH / 8; j++) {
            paged_store<BF16>(a, seg.m, h0 + h, 8 * j + 2 * t4, (o[rb][j][0] + o[rb][j][2]) * inv);
            paged_store<BF16>(a, seg.m, h0 + h, 8 * j + 2 * t4 + 1, (o[rb][j][1] + o[rb][j][3]) * inv);
          }
          if (t4 == 0) paged_store_lse<WEIGHTS>(a, seg.m, h0 + h, mx[rb], l[rb]);
        } else {
#pragma unroll
          for (int j = 0; j < DH / 8; j++)
            *reinterpret_cast<float2*>(state + h * DH + 8 * j + 2 * t4) =
                make_float2((o[rb][j][0] + o[rb][j][2]) * PagedP<BF16>::kDown,
                            (o[rb][j][1] + o[rb][j][3]) * PagedP<BF16>::kDown);
          if (t4 == 0) {
            state[srows * DH + h] = mx[rb];
            state[srows * DH + srows + h] = l[rb];
          }
        }
      }
      if (!all && !inside) {
        open[side] = seg;
        open_t[side] = f;
      }
      at += end - begin;
      next_pair(seg);
    }
    cp_async_wait<0>();
    // the last part of an open pair to arrive joins it.  (Arriving here, not where a
    // pair ends: a fence and an atomic in mid-stream stall the loads.)
    __syncwarp();
    int last = 0;
    if (lane < 2 && open_t[lane] >= 0) {
      const int p0 = cut.part_of(open_t[lane]), p1 = cut.part_of(open_t[lane] + open[lane].nt - 1);
      __threadfence();
      unsigned* arrived = a.counters + p0;  // a part begins at most one pair that it does not finish
      last = atomicAdd(arrived, 1u) == (unsigned)(p1 - p0);
      if (last) *arrived = 0;  // ready for the next call
      __threadfence();
    }
    const unsigned joins = __ballot_sync(0xffffffffu, last != 0);
#pragma unroll 1
    for (int side = 0; side < 2; side++) {
      if (!((joins >> side) & 1u)) continue;
      const PagedCursor p = open[side];
      const int hk = p.hv / a.chunks, h0 = hk * a.G + (p.hv % a.chunks) * ROWS;
      paged_join<DH, ROWS, BF16, WEIGHTS>(a, cut, open_t[side], p.nt, p.m, h0, min(ROWS, (hk + 1) * a.G - h0),
                                          reinterpret_cast<int*>(ring), 0, 1);
    }
  }
  if (!inside) return;

  // ---- a share inside one pair: the four warps' states -> one
  __syncthreads();
  const int hk = pair0.hv / a.chunks, h0 = hk * a.G + (pair0.hv % a.chunks) * ROWS;
  const int rows = min(ROWS, (hk + 1) * a.G - h0);
  const bool alone = t0 == pair0_t && t1 == pair0_t + pair0.nt;
  float* part = a.parts + 2 * c * kPagedWarps * sf;
  for (int e = tid; e < rows * DH; e += kPagedThreads) {
    const int h = e / DH;
    const float* st[kPagedWarps];
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPagedWarps; w++) {
      st[w] = reinterpret_cast<const float*>(paged_smem + w * (S * C::kStageBytes));
      m = fmaxf(m, st[w][srows * DH + h]);
    }
    const float ms = m == -INFINITY ? 0.0f : m;
    float acc = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kPagedWarps; w++) {
      const float lw = st[w][srows * DH + srows + h];
      if (lw == 0.0f) continue;  // an empty state's O was not written
      const float x = paged_ex2(st[w][srows * DH + h] - ms);
      acc = fmaf(x, st[w][e], acc);
      l = fmaf(x, lw, l);
    }
    if (alone) {
      paged_store<BF16>(a, pair0.m, h0 + h, e % DH, l == 0.0f ? 0.0f : acc / l);
      if (e % DH == 0) paged_store_lse<WEIGHTS>(a, pair0.m, h0 + h, m, l);
    } else {
      part[e] = acc;
      if (e % DH == 0) {
        part[srows * DH + h] = m;
        part[srows * DH + srows + h] = l;
      }
    }
  }
  if (alone) return;
  __syncthreads();
  if (tid == 0) {
    const int p0 = cut.part_of(pair0_t), p1 = cut.part_of(pair0_t + pair0.nt - 1);
    __threadfence();
    unsigned* arrived = a.counters + p0;
    s_last = atomicAdd(arrived, (unsigned)kPagedWarps) + kPagedWarps == (unsigned)(p1 - p0 + 1);
    if (s_last) *arrived = 0;
    __threadfence();
  }
  __syncthreads();
  if (s_last)  // the four warps take the rows in turn
    paged_join<DH, ROWS, BF16, WEIGHTS>(a, cut, pair0_t, pair0.nt, pair0.m, h0, rows, reinterpret_cast<int*>(ring), warp,
                                        kPagedWarps);
}

constexpr int kPagedWPT = 4;  // slots per thread

// weights_out[m][hk][j] = weights_in[m][hk][j] (0 for the new token's slot) +
// sum over the group's heads of 2^(score - lse2), the scores as the attention
// kernel left them; slot_pos of the new token's slot.  Slots past the end are
// not touched.  4 G + 8 bytes per slot, from L2 mostly: bound by its launch.
__global__ void __launch_bounds__(256) paged_weights_kernel(const PagedArgs a, const float* win, float* wout,
                                                            long long cap, int* slot_pos, const int* positions) {
  grid_dep_wait();  // launched while the attention kernel drains
  const int m = blockIdx.z, hk = blockIdx.y;
  const int n = paged_slots(a, m);
  const int old = n > 0 && a.k_new != nullptr ? n - 1 : n;
  const size_t at = ((size_t)m * a.Hkv + hk) * cap;
  const size_t h0 = (size_t)m * a.Hq + hk * a.G;
  const int j0 = blockIdx.x * (256 * kPagedWPT) + threadIdx.x;
  float w[kPagedWPT];
#pragma unroll
  for (int u = 0; u < kPagedWPT; u++) {
    const int j = j0 + 256 * u;
    w[u] = j < old ? win[at + j] : 0.0f;
  }
  for (int g = 0; g < a.G; g++) {
    const float ls = a.lse2[h0 + g];
    if (ls == -INFINITY) continue;  // a row that saw nothing
    const float* sc = a.scores + (h0 + g) * a.score_row;
#pragma unroll
    for (int u = 0; u < kPagedWPT; u++) {
      const int j = j0 + 256 * u;
      if (j < n) w[u] += paged_ex2(sc[j] - ls);
    }
  }
#pragma unroll
  for (int u = 0; u < kPagedWPT; u++) {
    const int j = j0 + 256 * u;
    if (j >= n) break;
    wout[at + j] = w[u];
    if (j >= old && slot_pos) slot_pos[at + j] = positions[m];
  }
}

// ------------------------------------------------------------------ host side
static int paged_chunks(int DH, int G) {
  const int rows = G <= 8 || DH == 256 ? 8 : 16;
  return (G + rows - 1) / rows;
}

static int paged_grid() { return 2 * sm_count(); }

static size_t paged_part_bytes(int DH, int G) {
  const int rows = G <= 8 || DH == 256 ? 8 : 16;
  return align_up((size_t)2 * kPagedWarps * paged_grid() * paged_state_floats(DH, G < rows ? G : rows) * sizeof(float),
                  256);
}

// Workspace: one counter per warp (zero between calls; a region of fixed size, so
// that calls of any shape may follow one another), partial states, and for the
// accumulated weights one log-sum-exp and score_row scores per query head.
size_t paged_counter_bytes() { return align_up((size_t)paged_grid() * kPagedWarps * sizeof(unsigned), 256); }

size_t paged_workspace_bytes(int M, int Hq, int Hkv, int DH, long long slots, bool weights) {
  const int G = Hq / Hkv;
  size_t b = paged_counter_bytes() + paged_part_bytes(DH, G);
  if (weights) b += align_up((size_t)M * Hq * sizeof(float), 256) + (size_t)M * Hq * align_up(slots, 4) * sizeof(float);
  return b;
}

template <int DH, int RB, bool BF16, bool WEIGHTS, bool PAGE16>
static cudaError_t launch_paged_t(PagedArgs a, cudaStream_t st) {
  // the deepest ring with which two CTAs share an SM; where that is no ring, one CTA
  const int lens = (2 * a.M + 1) * (int)sizeof(int);
  int per_sm = 2, fixed = 0;
  for (; per_sm > 0; per_sm--) {
    const int room = (per_sm == 2 ? 112 : 224) * 1024 - lens;
    a.stages = std::min(kPagedMaxStages, room / (kPagedWarps * PagedCfg<DH, RB>::kStageBytes));
    fixed = kPagedWarps * a.stages * PagedCfg<DH, RB>::kStageBytes;
    if (a.stages >= 2) break;
  }
  if (per_sm == 0) return cudaErrorInvalidValue;
  constexpr auto kern = attn_paged_kernel<DH, RB, BF16, WEIGHTS, PAGE16>;
  if (cudaError_t e = allow_smem<kern>(225 * 1024)) return e;
  kern<<<per_sm * sm_count(), kPagedThreads, fixed + lens, st>>>(a);
  return cudaGetLastError();
}

template <int DH, int RB>
static cudaError_t launch_paged_d(const PagedArgs& a, bool bf16, bool weights, cudaStream_t st) {
  auto by_page = [&](auto b, auto w) {
    constexpr bool B = decltype(b)::value, W = decltype(w)::value;
    return a.page_size % 16 == 0 ? launch_paged_t<DH, RB, B, W, true>(a, st)
                                 : launch_paged_t<DH, RB, B, W, false>(a, st);
  };
  using T = std::true_type;
  using F = std::false_type;
  if (bf16) return weights ? by_page(T(), T()) : by_page(T(), F());
  return weights ? by_page(F(), T()) : by_page(F(), F());
}

cudaError_t launch_attention_paged(PagedArgs a, int DH, bool bf16, void* ws, const float* win, float* wout,
                                   long long cap, int* slot_pos, const int* positions, cudaStream_t st) {
  const bool weights = wout != nullptr;
  a.chunks = paged_chunks(DH, a.G);
  a.Hv = a.Hkv * a.chunks;
  page_divisor(a.page_size, a.page_mul, a.page_shift);
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.slots + 256 * kPagedWPT - 1) / (256 * kPagedWPT)), a.Hkv, a.M);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_weights_kernel, (const PagedArgs)a, win, wout, cap, slot_pos, positions);
}

}  // namespace aria_q4
