// q4_paged.cuh -- the paged KV cache as its kernels see it.
//
// Keys and values live in pages of page_size slots; sequence m's slot j is row
// j % page_size of page table[m][j / page_size].  An entry of the table outside
// [0, num_pages) has no page: its slots are absent (never read, weight zero).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace aria_q4 {

constexpr int kPagedMaxSequences = 4096;  // of a call: their lengths and tile counts sit in shared memory

// A pair (sequence, head) of at most this many slots is not split when every
// pair has a CTA of its own; otherwise a CTA takes at least kPagedMinSlots.
constexpr int kPagedWholeSlots = 512;
constexpr int kPagedMinSlots = 128;

struct PagedArgs {
  int M, Hq, Hkv, G;        // sequences, query heads, key/value heads, Hq / Hkv
  int Hv, chunks;           // pairs per sequence: key/value heads x chunks of query heads
  const uint16_t* q;        // 16-bit floats; element strides throughout
  long long q_row, q_head;
  const uint16_t* k_pages;
  const uint16_t* v_pages;
  uint16_t* k_pages_w;      // the same pages, written only at the new token's slot
  uint16_t* v_pages_w;
  long long page_stride, slot_stride, head_stride;
  int num_pages, page_size;
  unsigned page_mul;        // slot / page_size = slot * page_mul >> page_shift
  int page_shift;
  const int* table;
  int table_stride, max_pages;
  const int* lens;          // slots in use before the call
  const uint16_t* k_new;    // the new token's rows (null: none is added)
  const uint16_t* v_new;
  long long new_row, new_head;
  float scale_log2;         // scale * log2(e)
  uint16_t* out;
  long long out_row, out_head;
  float* lse;               // [M][Hq], natural log; may be null
  long long slots;          // max_pages * page_size
  unsigned* counters;       // one per warp: arrivals at the pair that it begins and others finish
  float* parts;             // [warp][2]: states of the pairs that it shares at its start and at its end
  float* lse2;              // [M][Hq], log2 (accumulated weights only)
  float* scores;            // [M][Hq][score_row], log2 domain
  long long score_row;
  int stages;               // of every warp's ring
};

constexpr long long kEvictMaxSlots = 12 << 20;  // of a sequence: a bit per slot sits in shared memory

struct EvictArgs {
  int M, Hkv;
  uint16_t* k_pages;
  uint16_t* v_pages;
  long long page_stride, slot_stride, head_stride;
  int num_pages, page_size;
  unsigned page_mul;         // as above
  int page_shift;
  const int* table;
  int table_stride, max_pages;
  const int* lens;
  long long slots;           // the table's width in slots
  const float* weights_in;   // [M][Hkv][cap]; the outputs may be the inputs
  float* weights_out;
  const int* pos_in;
  int* pos_out;
  long long cap;
  const int* next_pos;       // [M] position of each sequence's next token
  int* lens_out;             // may be null
  int keep, recent, sinks;
  int row_bytes;             // of one K row
  int cluster;
  int bit_words;             // words of a CTA's bits (a multiple of 4)
  int* lists;                // [M * Hkv][2][list_len]: holes, survivors that move
  long long list_len;
  int* moves;                // [M * Hkv]: entries of a row's lists
  int fused;                 // the rows are moved by the kernel that chooses them
  int segment;               // moves per CTA of the kernel that moves them
};

// slot / page_size = slot * mul >> shift, exact for slots below 2^31: with
// 2^(l-1) < d <= 2^l, M = ceil(2^(31+l) / d) fits 32 bits and M d - 2^(31+l) < d
inline void page_divisor(int page_size, unsigned& mul, int& shift) {
  int l = 0;
  while ((1LL << l) < page_size) l++;
  shift = 31 + l;
  mul = (unsigned)(((1ULL << shift) + page_size - 1) / page_size);
}

// Slots sequence m attends over: those in use, and the new token's.  A new
// token without room in the table leaves the sequence with none.
__device__ __forceinline__ int paged_slots(const PagedArgs& a, int m) {
  const int n = max(a.lens[m], 0);
  if (a.k_new != nullptr) return n < a.slots ? n + 1 : 0;
  return (int)min((long long)n, a.slots);
}

template <bool BF16>
__device__ __forceinline__ void paged_store(const PagedArgs& a, int m, int h, int d, float v) {
  const long long at = (long long)m * a.out_row + (long long)h * a.out_head + d;
  if (BF16)
    reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(v);
}

// mx: the row's maximum in the log2 domain, sum: of 2^(s - mx), 0 for a row that saw nothing
template <bool WEIGHTS>
__device__ __forceinline__ void paged_store_lse(const PagedArgs& a, int m, int h, float mx, float sum) {
  const float l2 = sum == 0.0f ? -INFINITY : mx + log2f(sum);
  if (a.lse) a.lse[(size_t)m * a.Hq + h] = l2 * 0.69314718055994531f;
  if (WEIGHTS) a.lse2[(size_t)m * a.Hq + h] = l2;
}

}  // namespace aria_q4
