// prompt_weights.cu -- the attention weight every position of a prompt has received,
// on the 5th-generation tensor cores (tcgen05, sm_100a).
//
// After the prompt's causal attention (its log-sum-exp rows are kept), for key/value
// head hk of G query heads and key position s:
//   w[b][hk][s] = sum over the group's heads h and queries t >= max(s, first) of
//                 exp(scale q[b][t][h] . k[b][s][hk] - lse[b][h][t])
// the start of the running sums that eviction ranks positions by.
//
// The product is computed transposed, S = K Q^T: a block of 128 keys is the A operand
// (TMEM lanes = keys) and stays in shared memory while the blocks of 128 queries of
// every head of the group stream past as B.  A thread then owns one key and adds up
// its row of S in registers: no reduction across threads, nothing but the finished
// sums leaves the SM.  Per 128 x 128 block: 2 dh / 128 MMA cycles x 128 (256 at
// dh = 64) against 16384 exponentials at 16 a cycle (1024 cycles), so the exponential
// unit is the bound: it is 85% busy over 2 x 8190 positions x 32 heads of 128 (8 groups of
// 4, queries from 2047 on: 596 us, 680 to 690 once the power limit holds the clock at 1.5
// to 1.7 GHz), 65% over 4 x 2048 x 14 heads of 64, where the start and the items' ends
// count.  At dh = 64 one pair in eight goes through a polynomial on the multiply-add pipe
// instead (the longer size with heads of 64: 558 -> 520 us; two pairs: 531); at 128 the
// added instructions lowered the clock by more than they saved (597 -> 619).
//
// Persistent, one CTA per SM; an item is (sequence, key/value head, key block) or, where
// those are few, a part of its query blocks (the last part to finish adds the parts' sums
// in order); the first blocks (most queries) first, dealt out in alternating directions.  Twenty warps:
//   warp 0      TMA producer: K blocks (two buffers), Q blocks into a ring
//   warp 1      TMEM allocator and single-thread MMA issuer
//   warps 2-17  sums: a warp per TMEM lane quadrant and S buffer, so that the four
//               warps of a sub-partition are at different blocks and keep its
//               exponential unit busy through one another's waits.  (Four warps per
//               block, a quarter of the queries each: 55 us at 4 x 2048 x 14 heads,
//               the same call repeated; two warps: 70 us, the unit 40% busy; so: 41 us,
//               44 with other inputs each time.)
//   warp 18     lse rows of the query blocks -> shared memory, negated, in the log2 domain;
//               -inf for queries before `first` or past the end, whose terms vanish, and
//               for those whose lse is -inf, with a word by which the block's scores are
//               looked at first (theirs need not be finite)
//   warp 19     adds an item's four sums per key and stores them
// Every wait is bounded (one second for the MMA issuer, two for the others; an abort
// flag; the code in this unit's g_device_error).
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "q4_common.cuh"
#include "q4_status.cuh"
#include "q4_tcgen05.cuh"

namespace aria_q4 {

constexpr int kPwSumWarps = 16;
constexpr int kPwThreads = (4 + kPwSumWarps) * 32;
constexpr int kPwB = 128;     // keys per item, queries per block
constexpr int kPwS = 4;       // S buffers (128 TMEM columns each) and lse buffers

struct PromptArgs {
  int B, T, Hkv, G, first;
  float scale_log2;
  const float* lse;           // [B][Hq][T]
  float* w;                   // element strides w_seq, w_head
  long long w_seq, w_head;
  int n_kt;                   // key blocks of a sequence
  int splits;                 // items per (sequence, key/value head, key block)
  float* parts;               // [item][128] sums, and [item / splits] arrivals (zero between
  unsigned* arrived;          // calls), where an item is a part of a key block's sums
  unsigned long long wait_ns;
};

template <int DH>
struct PromptSmem {
  static constexpr int kTile = kPwB * DH * 2;
  static constexpr int kNQ = DH == 64 ? 6 : 4;              // Q ring stages
  static constexpr int kKOff = 0;                           // [2]
  static constexpr int kQOff = 2 * kTile;                   // [kNQ]
  static constexpr int kLseOff = kQOff + kNQ * kTile;       // [kPwS][128] f32
  static constexpr int kSumOff = kLseOff + kPwS * kPwB * 4;  // [2 items][kPwS][128] f32: the buffers' sums
  static constexpr int kBarOff = kSumOff + 2 * kPwS * kPwB * 4;
  static constexpr int kBytes = kBarOff + 512 + 1024;
};

struct PromptItem {
  int seq, hk, kt, q0, nq;  // query blocks q0 .. q0 + nq - 1 of each head, head by head:
  int lo, hi;               // of these G nq blocks, this item's
  int index;                // of the item
};
// Item of CTA blockIdx.x in round t / gridDim.x (t = blockIdx.x + round * gridDim.x):
// odd rounds run backwards, so that no CTA has the longer item of every round.
__device__ __forceinline__ PromptItem prompt_item(const PromptArgs& a, int t, int n_items) {
  const int g = (int)gridDim.x, round = t / g;
  if (round & 1) {
    const int size = min(g, n_items - round * g);  // the last round may be short
    t = round * g + (size - 1 - t % g);
  }
  const int bh = a.B * a.Hkv;
  int base = t, split = 0;
  if (a.splits > 1) {
    base = t / a.splits;
    split = t - base * a.splits;
  }
  PromptItem r;
  r.index = t;
  r.kt = base / bh;
  base -= r.kt * bh;
  r.seq = base / a.Hkv;
  r.hk = base - r.seq * a.Hkv;
  r.q0 = max(r.kt, a.first / kPwB);
  r.nq = max(0, a.n_kt - r.q0);
  r.lo = 0;
  r.hi = a.G * r.nq;
  if (a.splits > 1) {
    const long long blocks = r.hi;
    r.lo = (int)(blocks * split / a.splits);
    r.hi = (int)(blocks * (split + 1) / a.splits);
  }
  return r;
}

// Two f32 values in a register pair, and arithmetic on both in one instruction.
__device__ __forceinline__ uint64_t pack2(uint32_t x, uint32_t y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x of two values on the multiply-add pipe: x = n + f with n an integer and |f| <= 1/2
// (n from the low bits of x + 1.5 2^23), a polynomial in f of degree 5 whose coefficients
// minimise the largest relative error on that interval (Lawson's iteration; 2.3e-7
// evaluated in f32), times 2^n.  x below -126 gives 0 (-inf does, for masked queries), x
// from 127.5 on inf.  NaN stays NaN because 2^n is a factor: added to the exponent, n made
// a large finite number of the NaN's bits.
__device__ __forceinline__ uint64_t both(float x) { return pack2(__float_as_uint(x), __float_as_uint(x)); }
__device__ __forceinline__ void exp2_poly2(float& x, float& y) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(128.0f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(128.0f));
  const uint64_t v = pack2(__float_as_uint(x), __float_as_uint(y));
  const uint64_t t = add2(v, both(12582912.0f));
  const uint64_t f = fma2(add2(t, both(-12582912.0f)), both(-1.0f), v);
  uint64_t p = fma2(both(1.3276472e-3f), f, both(9.675541e-3f));
  p = fma2(p, f, both(5.5507131e-2f));
  p = fma2(p, f, both(2.402212e-1f));
  p = fma2(p, f, both(6.9314694e-1f));
  p = fma2(p, f, both(1.0000001f));
  float p0, p1, t0, t1;
  unpack2(t, t0, t1);
  unpack2(mul2(p, pack2((__float_as_uint(t0) << 23) + 0x3f800000u, (__float_as_uint(t1) << 23) + 0x3f800000u)), p0, p1);
  x = x < -126.0f ? 0.0f : p0;
  y = y < -126.0f ? 0.0f : p1;
}

// The terms of one block of queries, each taken by selection: those from cmin on that saw
// something.  neg_lse: the block's.  (Beside the unrolled loop, not in it: a test there for
// blocks that hardly occur took 46 us to 51 at 4 x 2048 x 14 heads.)
__device__ __forceinline__ uint64_t prompt_selected(uint32_t s_col, const float* neg_lse, int cmin, float scale_log2) {
  float sum = 0.0f;
#pragma unroll 1
  for (int c = 0; c < kPwB; c += 16) {
    uint32_t sv[16];
    tc::tmem_ld_32x32b_x16(s_col + c, sv);
    tc::tmem_ld_wait();
    tc::reg_tie(sv);
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const float l = neg_lse[c + e];
      const float p = tc::ex2_approx(fmaf(__uint_as_float(sv[e]), scale_log2, l));
      sum += c + e >= cmin && l != -INFINITY ? p : 0.0f;
    }
  }
  return pack2(__float_as_uint(sum), 0u);
}

template <int DH, bool BF16>
__global__ void __launch_bounds__(kPwThreads, 1)
    prompt_weights_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                          const PromptArgs a) {
  using L = PromptSmem<DH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);  // [2]
  uint64_t* k_empty = k_full + 2;                                     // [2] MMA commit after the item's last block
  uint64_t* q_full = k_empty + 2;                                     // [kNQ]
  uint64_t* q_empty = q_full + L::kNQ;                                // [kNQ] MMA commit
  uint64_t* s_full = q_empty + L::kNQ;                                // [kPwS] MMA commit and lse warp
  uint64_t* s_empty = s_full + kPwS;                                  // [kPwS] 4 summing warps: S read
  uint64_t* l_empty = s_empty + kPwS;                                 // [kPwS] 4 summing warps: lse read
  uint64_t* p_full = l_empty + kPwS;                                  // [2] all summing warps: an item's sums
  uint64_t* p_empty = p_full + 2;                                     // [2] warp 19
  uint64_t* mma_drain = p_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_drain + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  int* lse_gaps = abort_flag + 1;  // [kPwS] whether some query of the block saw nothing
  float* lse_s = reinterpret_cast<float*>(smem + L::kLseOff);
  float* part_sum = reinterpret_cast<float*>(smem + L::kSumOff);
  auto give_up = [&](int wait_result, int code) {
    if (wait_result == tc::kWaitTimeout) tc::record_error(code);
    atomicExch(abort_flag, 1);
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_items = a.n_kt * a.B * a.Hkv * a.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; s++) {
      tc::mbar_init(&k_full[s], 1);
      tc::mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < L::kNQ; s++) {
      tc::mbar_init(&q_full[s], 1);
      tc::mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < kPwS; s++) {
      tc::mbar_init(&s_full[s], 2);
      tc::mbar_init(&s_empty[s], 4);
      tc::mbar_init(&l_empty[s], 4);
    }
    for (int s = 0; s < 2; s++) {
      tc::mbar_init(&p_full[s], kPwSumWarps);
      tc::mbar_init(&p_empty[s], 1);
    }
    tc::mbar_init(mma_drain, 1);
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tc::prefetch_tmap(&tm_q);
    tc::prefetch_tmap(&tm_k);
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Every role walks the same items and query blocks; phases follow the CTA-wide
  // block counter g and item counter it.
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int g = 0, it = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const int w = tc::mbar_wait_or_abort(bar, parity, 2 * a.wait_ns, abort_flag);
        if (w != tc::kWaitOk) {
          give_up(w, tc::kErrTimeoutEmpty);
          ok = false;
        }
        return ok;
      };
      for (int t = blockIdx.x; t < n_items && ok; t += gridDim.x) {
        const PromptItem im = prompt_item(a, t, n_items);
        if (im.lo >= im.hi) continue;
        const int kb = it & 1;
        if (it >= 2 && !wait(&k_empty[kb], ((it >> 1) - 1) & 1)) break;
        tc::mbar_arrive_expect_tx(&k_full[kb], L::kTile);
#pragma unroll
        for (int c = 0; c < DH / 64; c++)
          tc::tma_load_4d(smem + L::kKOff + kb * L::kTile + c * (kPwB * 128), &tm_k, 64 * c, im.hk, im.kt * kPwB,
                          im.seq, &k_full[kb]);
        it++;
        int h = im.lo / im.nq, qb = im.lo % im.nq;
        for (int j = im.lo; j < im.hi; j++, g++) {
          const int s = g % L::kNQ, use = g / L::kNQ;
          if (use >= 1 && !wait(&q_empty[s], (use - 1) & 1)) break;
          tc::mbar_arrive_expect_tx(&q_full[s], L::kTile);
#pragma unroll
          for (int c = 0; c < DH / 64; c++)
            tc::tma_load_4d(smem + L::kQOff + s * L::kTile + c * (kPwB * 128), &tm_q, 64 * c, im.hk * a.G + h,
                            (im.q0 + qb) * kPwB, im.seq, &q_full[s]);
          if (++qb == im.nq) {
            qb = 0;
            h++;
          }
        }
      }
      // no copy into shared memory may be in flight when the CTA exits
      for (int i = it > 2 ? it - 2 : 0; i < it; i++) tc::mbar_wait(&k_full[i & 1], (i >> 1) & 1);
      for (int i = g > L::kNQ ? g - L::kNQ : 0; i < g; i++) tc::mbar_wait(&q_full[i % L::kNQ], (i / L::kNQ) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = tc::idesc_f16_f32(128, kPwB) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        const int w = tc::mbar_wait_or_abort(bar, parity, a.wait_ns, abort_flag);
        if (w != tc::kWaitOk) {
          give_up(w, code);
          ok = false;
        }
        return ok;
      };
      int g = 0, it = 0;
      for (int t = blockIdx.x; t < n_items && ok; t += gridDim.x) {
        const PromptItem im = prompt_item(a, t, n_items);
        if (im.lo >= im.hi) continue;
        const int kb = it & 1;
        if (!wait(&k_full[kb], (it >> 1) & 1, tc::kErrTimeoutFull)) break;
        const uint32_t ks = tc::smem_u32(smem + L::kKOff + kb * L::kTile);
        const int blocks = im.hi - im.lo;
        for (int j = 0; j < blocks; j++, g++) {
          const int s = g % L::kNQ, b = g % kPwS;
          if (!wait(&q_full[s], (g / L::kNQ) & 1, tc::kErrTimeoutFull)) break;
          if (g >= kPwS && !wait(&s_empty[b], ((g / kPwS) - 1) & 1, tc::kErrTimeoutAccum)) break;
          tc::tc_fence_after();
          const uint32_t qs = tc::smem_u32(smem + L::kQOff + s * L::kTile);
#pragma unroll
          for (int kk = 0; kk < DH / 16; kk++)
            tc::umma_f16(tmem_base + (uint32_t)(b * kPwB),
                         tc::sdesc_k_sw128(ks + (kk >> 2) * (kPwB * 128) + (kk & 3) * 32),
                         tc::sdesc_k_sw128(qs + (kk >> 2) * (kPwB * 128) + (kk & 3) * 32), idesc, kk > 0 ? 1u : 0u);
          tc::umma_commit(&s_full[b]);
          tc::umma_commit(&q_empty[s]);
          if (j == blocks - 1) tc::umma_commit(&k_empty[kb]);
        }
        it++;
      }
      // no MMA of this thread may still write tensor memory when it is freed, nor arrive at a
      // barrier of a CTA that has left.  (The sums wait for every product, but a warp that gives
      // up after the last one was issued takes the others along.)
      tc::umma_commit(mma_drain);
      tc::mbar_wait(mma_drain, 0);
    }
  } else if (warp < 2 + kPwSumWarps) {
    // ------------------------------------------------------------ sums
    const int qd = warp & 3;           // TMEM lane quadrant
    const int b = (warp - 2) >> 2;     // S buffer: blocks g = b, b + kPwS, ...
    const int r = qd * 32 + lane;      // key of the block = TMEM lane
    const uint32_t s_col = tmem_base + ((uint32_t)(qd * 32) << 16) + (uint32_t)(b * kPwB);
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
      const int w = tc::mbar_wait_or_abort(bar, parity, 2 * a.wait_ns, abort_flag);
      if (__all_sync(0xffffffffu, w == tc::kWaitOk)) return true;
      const bool any_timeout = __any_sync(0xffffffffu, w == tc::kWaitTimeout);
      if (lane == 0) give_up(any_timeout ? tc::kWaitTimeout : tc::kWaitAborted, code);
      ok = false;
      return false;
    };
    int g0 = 0, it = 0;    // first block and number of the item
    uint32_t uses = 0;     // blocks of this buffer so far
    const uint64_t scale2 = pack2(__float_as_uint(a.scale_log2), __float_as_uint(a.scale_log2));
    for (int t = blockIdx.x; t < n_items && ok; t += gridDim.x, it++) {
      const PromptItem im = prompt_item(a, t, n_items);
      const int key = im.kt * kPwB + r, blocks = im.hi - im.lo;
      const int masked = max(im.kt * kPwB + kPwB - 1, a.first);  // from this query on nothing is left out
      uint64_t sum[2] = {0, 0};  // four running sums
      int j = (b - g0) & (kPwS - 1);
      int qb = im.nq > 0 ? (im.lo + j) % im.nq : 0;  // query block of the head
      for (; j < blocks; j += kPwS, uses++) {
        if (!wait(&s_full[b], uses & 1, tc::kErrTimeoutFull)) break;
        tc::tc_fence_after();
        uint32_t sv[2][16];
        tc::tmem_ld_32x32b_x16(s_col, sv[0]);
        const int q0 = (im.q0 + qb) * kPwB;
        for (qb += kPwS; qb >= im.nq;) qb -= im.nq;
        if (lse_gaps[b] != 0) {  // queries that saw nothing: their scores need not be finite
          tc::tmem_ld_wait();
          tc::reg_tie(sv[0]);
          sum[0] = add2(sum[0], prompt_selected(s_col, lse_s + b * kPwB, max(key, a.first) - q0, a.scale_log2));
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            tc::mbar_arrive(&s_empty[b]);
            tc::mbar_arrive(&l_empty[b]);
          }
          continue;
        }
#pragma unroll
        for (int c = 0; c < 8; c++) {
          tc::tmem_ld_wait();
          tc::reg_tie(sv[c & 1]);
          if (c < 7) {
            tc::tmem_ld_32x32b_x16(s_col + 16 * (c + 1), sv[(c + 1) & 1]);
          } else {  // the scores are in registers: the next product may begin
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s_empty[b]);
          }
          const ulonglong2* ls = reinterpret_cast<const ulonglong2*>(lse_s + b * kPwB + c * 16);
          const int qc = q0 + c * 16;
          if (qc < masked) {
            // queries before the key or before `first` are left out by selection, so that
            // whatever their rows hold (a NaN too) does not reach the sums
            const int cmin = max(key, a.first) - qc;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const ulonglong2 l4 = ls[e >> 2];  // -lse of four queries
              const uint32_t* s4 = &sv[c & 1][e];
              float p0, p1, p2, p3;
              unpack2(fma2(pack2(s4[0], s4[1]), scale2, l4.x), p0, p1);
              unpack2(fma2(pack2(s4[2], s4[3]), scale2, l4.y), p2, p3);
              p0 = tc::ex2_approx(p0);
              p1 = tc::ex2_approx(p1);
              p2 = tc::ex2_approx(p2);
              p3 = tc::ex2_approx(p3);
              p0 = e >= cmin ? p0 : 0.0f;
              p1 = e + 1 >= cmin ? p1 : 0.0f;
              p2 = e + 2 >= cmin ? p2 : 0.0f;
              p3 = e + 3 >= cmin ? p3 : 0.0f;
              sum[0] = add2(sum[0], pack2(__float_as_uint(p0), __float_as_uint(p1)));
              sum[1] = add2(sum[1], pack2(__float_as_uint(p2), __float_as_uint(p3)));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const ulonglong2 l4 = ls[e >> 2];  // -lse of four queries
              const uint32_t* s4 = &sv[c & 1][e];
              float p0, p1, p2, p3;
              unpack2(fma2(pack2(s4[0], s4[1]), scale2, l4.x), p0, p1);
              unpack2(fma2(pack2(s4[2], s4[3]), scale2, l4.y), p2, p3);
              p0 = tc::ex2_approx(p0);
              p1 = tc::ex2_approx(p1);
              if (DH == 64 && e == 0) {
                exp2_poly2(p2, p3);
              } else {
                p2 = tc::ex2_approx(p2);
                p3 = tc::ex2_approx(p3);
              }
              sum[0] = add2(sum[0], pack2(__float_as_uint(p0), __float_as_uint(p1)));
              sum[1] = add2(sum[1], pack2(__float_as_uint(p2), __float_as_uint(p3)));
            }
          }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&l_empty[b]);
      }
      if (!ok) break;
      g0 += blocks;
      if (it >= 2 && !wait(&p_empty[it & 1], ((it >> 1) - 1) & 1, tc::kErrTimeoutEmpty)) break;
      float s0, s1, s2, s3;
      unpack2(sum[0], s0, s1);
      unpack2(sum[1], s2, s3);
      part_sum[((it & 1) * kPwS + b) * kPwB + r] = (s0 + s1) + (s2 + s3);
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[it & 1]);
    }
  } else if (warp == 3 + kPwSumWarps) {
    // ------------------------------------------------------------ an item's sums -> output
    int it = 0;
    for (int t = blockIdx.x; t < n_items; t += gridDim.x, it++) {
      const PromptItem im = prompt_item(a, t, n_items);
      const int w = tc::mbar_wait_or_abort(&p_full[it & 1], (it >> 1) & 1, 2 * a.wait_ns, abort_flag);
      if (!__all_sync(0xffffffffu, w == tc::kWaitOk)) {
        if (lane == 0) give_up(w, tc::kErrTimeoutFull);
        break;
      }
      const float* ps = part_sum + (it & 1) * kPwS * kPwB;
#pragma unroll
      for (int u = 0; u < kPwB / 32; u++) {
        const int r = 32 * u + lane, key = im.kt * kPwB + r;
        const float sum = (ps[r] + ps[kPwB + r]) + (ps[2 * kPwB + r] + ps[3 * kPwB + r]);
        if (a.splits > 1)
          a.parts[(size_t)im.index * kPwB + r] = sum;
        else if (key < a.T)
          a.w[(long long)im.seq * a.w_seq + (long long)im.hk * a.w_head + key] = sum;
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_empty[it & 1]);
      if (a.splits > 1) {  // the key block's last item adds all of them, in order
        int last = 0;
        if (lane == 0) {
          __threadfence();
          unsigned* arrived = a.arrived + im.index / a.splits;
          last = atomicAdd(arrived, 1u) == (unsigned)(a.splits - 1);
          if (last) *arrived = 0;  // ready for the next call
          __threadfence();
        }
        if (__shfl_sync(0xffffffffu, last, 0)) {
          const float* first = a.parts + (size_t)(im.index - im.index % a.splits) * kPwB;
#pragma unroll
          for (int u = 0; u < kPwB / 32; u++) {
            const int r = 32 * u + lane, key = im.kt * kPwB + r;
            float sum = 0.0f;
            for (int k = 0; k < a.splits; k++) sum += __ldcg(first + (size_t)k * kPwB + r);
            if (key < a.T) a.w[(long long)im.seq * a.w_seq + (long long)im.hk * a.w_head + key] = sum;
          }
        }
      }
    }
  } else if (warp == 2 + kPwSumWarps) {
    // ------------------------------------------------------------ lse rows
    // (a block's rows are fetched while the one before it waits for its buffer; which rows
    // they are is worked out one block earlier still)
    int t = blockIdx.x, j = 0, h = 0, qb = 0;
    PromptItem im;
    const float* row = nullptr;  // of block j
    auto begin = [&]() {         // the first block of item t, or of the first one after it that has any
      for (; t < n_items; t += gridDim.x) {
        im = prompt_item(a, t, n_items);
        if (im.lo < im.hi) {
          j = im.lo;
          h = im.lo / im.nq;
          qb = im.lo - h * im.nq;
          row = a.lse + ((size_t)im.seq * a.Hkv * a.G + im.hk * a.G + h) * a.T;
          return;
        }
      }
    };
    auto advance = [&]() {
      if (t >= n_items) return;
      if (++j == im.hi) {
        t += gridDim.x;
        begin();
      } else if (++qb == im.nq) {
        qb = 0;
        row += a.T;
      }
    };
    float next[4];
    auto fetch = [&]() {
      if (t >= n_items) return;
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int q = (im.q0 + qb) * kPwB + 32 * u + lane;
        next[u] = q < a.T && q >= a.first ? row[q] : INFINITY;
      }
    };
    begin();
    bool more = t < n_items;
    fetch();
    advance();
    for (int g = 0; more; g++) {
      const int b = g % kPwS;
      float v[4];
      bool gap = false;
#pragma unroll
      for (int u = 0; u < 4; u++) {
        v[u] = next[u] * -1.4426950408889634f;
        gap |= v[u] == INFINITY;  // a row that saw nothing gives nothing
        if (v[u] == INFINITY) v[u] = -INFINITY;
      }
      gap = __any_sync(0xffffffffu, gap);
      more = t < n_items;
      fetch();
      if (g >= kPwS) {
        const int w = tc::mbar_wait_or_abort(&l_empty[b], ((g / kPwS) - 1) & 1, 2 * a.wait_ns, abort_flag);
        if (!__all_sync(0xffffffffu, w == tc::kWaitOk)) {
          if (lane == 0) give_up(w, tc::kErrTimeoutEmpty);
          break;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; u++) lse_s[b * kPwB + 32 * u + lane] = v[u];
      if (lane == 0) lse_gaps[b] = gap;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&s_full[b]);
      advance();
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ host side
typedef CUresult (*PromptEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static PromptEncodeFn prompt_encode_fn() {
  static PromptEncodeFn fn = []() -> PromptEncodeFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<PromptEncodeFn>(p);
  }();
  return fn;
}

// {DH, H, T, B} view, boxes of 128 positions x 64 columns of one head
static bool prompt_tmap(CUtensorMap* tm, const void* base, bool bf16, int DH, int H, int T, int B, long long s_head,
                        long long s_pos, long long s_seq) {
  PromptEncodeFn enc = prompt_encode_fn();
  if (!enc) return false;
  const cuuint64_t dim[4] = {(cuuint64_t)DH, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  const cuuint64_t str[3] = {(cuuint64_t)s_head * 2, (cuuint64_t)s_pos * 2, (cuuint64_t)s_seq * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)kPwB, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(base), dim, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DH, bool BF16>
static cudaError_t launch_prompt_t(const PromptArgs& a, const CUtensorMap& tq, const CUtensorMap& tk,
                                   cudaStream_t st) {
  using L = PromptSmem<DH>;
  constexpr auto kern = prompt_weights_kernel<DH, BF16>;
  if (cudaError_t e = allow_smem<kern>(L::kBytes)) return e;
  const int sms = sm_count();
  const int items = a.n_kt * a.B * a.Hkv * a.splits;
  kern<<<items < sms ? items : sms, kPwThreads, L::kBytes, st>>>(tq, tk, a);
  return cudaGetLastError();
}

// Parts that a key block's sums are cut into.  A part costs about as much as 4 blocks
// (its K block, an empty pipeline, the join), so sums stay whole unless the longest is
// more than twice an SM's share of all blocks, or 16: then the parts are one and a half
// such shares.  (One head of 8192 positions, 64 key blocks of 64 to 1: 43 us uncut, 21
// to 25 cut; 14 heads of 2048, 16 blocks at most: 17 us uncut, 26 cut in two.)
constexpr int kPwMaxCut = 1024;  // key blocks that may be cut: a fixed number of counters
static int prompt_splits(int B, int T, int Hkv, int G, int first) {
  const long long n_kt = (T + kPwB - 1) / kPwB, base = n_kt * B * Hkv;
  const long long f0 = std::min<long long>(first / kPwB, n_kt), n = n_kt - f0, longest = G * n;
  if (base > kPwMaxCut) return 1;
  const long long all = (long long)B * Hkv * G * (f0 * n + n * (n + 1) / 2);
  const long long share = std::max(8LL, all / sm_count());
  if (longest <= 2 * share) return 1;
  return (int)((2 * longest + 3 * share - 1) / (3 * share));
}

size_t prompt_counter_bytes() { return kPwMaxCut * sizeof(unsigned); }

size_t prompt_workspace_bytes(int B, int T, int Hkv, int G, int first) {
  const int splits = prompt_splits(B, T, Hkv, G, first);
  if (splits == 1) return 0;
  const size_t base = (size_t)((T + kPwB - 1) / kPwB) * B * Hkv;
  return prompt_counter_bytes() + base * splits * kPwB * sizeof(float);
}

cudaError_t launch_prompt_weights(const void* q, const void* k, bool bf16, int DH, long long q_seq, long long q_pos,
                                  long long q_head, long long k_seq, long long k_pos, long long k_head, int B, int T,
                                  int Hkv, int G, int first, float scale, const float* lse, float* w, long long w_seq,
                                  long long w_head, void* ws, cudaStream_t st) {
  CUtensorMap tq, tk;
  if (!prompt_tmap(&tq, q, bf16, DH, Hkv * G, T, B, q_head, q_pos, q_seq) ||
      !prompt_tmap(&tk, k, bf16, DH, Hkv, T, B, k_head, k_pos, k_seq))
    return cudaErrorInvalidValue;
  PromptArgs a;
  a.B = B; a.T = T; a.Hkv = Hkv; a.G = G; a.first = first;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.lse = lse;
  a.w = w; a.w_seq = w_seq; a.w_head = w_head;
  a.n_kt = (T + kPwB - 1) / kPwB;
  a.splits = prompt_splits(B, T, Hkv, G, first);
  a.arrived = (unsigned*)ws;
  a.parts = (float*)((uint8_t*)ws + prompt_counter_bytes());
  a.wait_ns = tc::kWaitLimitNs;
  if (DH == 64) return bf16 ? launch_prompt_t<64, true>(a, tq, tk, st) : launch_prompt_t<64, false>(a, tq, tk, st);
  if (DH == 128) return bf16 ? launch_prompt_t<128, true>(a, tq, tk, st) : launch_prompt_t<128, false>(a, tq, tk, st);
  return cudaErrorInvalidValue;
}

// Reads and clears this unit's device error flag (synchronous).
int prompt_take_device_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, tc::g_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(tc::g_device_error, &zero, sizeof(int));
  return v;
}

}  // namespace aria_q4
