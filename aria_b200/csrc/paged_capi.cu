// paged_capi.cu -- extern "C" entry points of the paged KV cache and of the logits
// (declared in include/aria_q4.h): argument checks and status codes; the kernels
// live in attn_paged.cu, prompt_weights.cu, cache_evict.cu and logits.cu.
#include <initializer_list>

#include "../../include/aria_q4.h"
#include "q4_common.cuh"
#include "q4_logits.cuh"
#include "q4_paged.cuh"
#include "q4_status.cuh"

namespace aria_q4 {
size_t paged_counter_bytes();
size_t prompt_counter_bytes();
size_t paged_workspace_bytes(int M, int Hq, int Hkv, int DH, long long slots, bool weights);
cudaError_t launch_attention_paged(PagedArgs a, int DH, bool bf16, void* ws, const float* win, float* wout,
                                   long long cap, int* slot_pos, const int* positions, cudaStream_t st);
cudaError_t launch_prompt_weights(const void* q, const void* k, bool bf16, int DH, long long q_seq, long long q_pos,
                                  long long q_head, long long k_seq, long long k_pos, long long k_head, int B, int T,
                                  int Hkv, int G, int first, float scale, const float* lse, float* w, long long w_seq,
                                  long long w_head, void* ws, cudaStream_t st);
size_t prompt_workspace_bytes(int B, int T, int Hkv, int G, int first);
size_t evict_workspace_bytes(int M, int Hkv, long long slots, int keep);
cudaError_t launch_cache_evict(EvictArgs a, void* ws, cudaStream_t st);
size_t logits_workspace_bytes(int M);
cudaError_t launch_logits_adjust(LogitArgs a, int din, int dout, void* ws, cudaStream_t st);
}  // namespace aria_q4

using namespace aria_q4;

static const long long kMaxSlots = 0x7fffff00;   // of one sequence

// whether every pointer is a multiple of n bytes (its element's size; NULL is)
static bool elements_aligned(size_t n, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if ((uintptr_t)p % n) return false;
  return true;
}

static int check_kv(const aria_paged_kv* kv, int M, long long* slots) {
  if (!kv || M < 0) return ARIA_Q4_EINVAL;
  if (kv->kv_heads <= 0 || kv->page_size <= 0 || kv->max_pages <= 0 || kv->num_pages < 0 ||
      kv->table_stride < kv->max_pages)
    return ARIA_Q4_EINVAL;
  if (kv->dtype != ARIA_Q4_F16 && kv->dtype != ARIA_Q4_BF16) return ARIA_Q4_EINVAL;
  const int dh = kv->head_dim;
  if (dh != 32 && dh != 64 && dh != 128 && dh != 256) return ARIA_Q4_EUNSUPPORTED;
  if (M > kPagedMaxSequences || kv->kv_heads > 65535) return ARIA_Q4_EUNSUPPORTED;  // (heads: a grid dimension)
  *slots = (long long)kv->page_size * kv->max_pages;
  if (*slots > kMaxSlots || (long long)M * ((*slots + 15) / 16) > 0x7fffffffLL) return ARIA_Q4_ESIZE;
  if (kv->page_stride % 8 || kv->slot_stride % 8 || kv->head_stride % 8) return ARIA_Q4_EALIGN;
  if (M == 0) return ARIA_Q4_OK;
  if (!kv->k_pages || !kv->v_pages || !kv->block_table || !kv->lens) return ARIA_Q4_EINVAL;
  if (!aligned16(kv->k_pages) || !aligned16(kv->v_pages) || !elements_aligned(4, {kv->block_table, kv->lens}))
    return ARIA_Q4_EALIGN;
  return ARIA_Q4_OK;
}

// the key blocks of all sequences and heads, and the query blocks of a key block, count in 31 bits
static bool prompt_blocks_fit(int B, int T, int heads, int kv_heads) {
  const long long blocks = ((long long)T + 127) / 128, most = 0x7fffffffLL / 1024;
  return blocks <= most / kv_heads / B && blocks <= 0x7fffffffLL / heads;
}

extern "C" {

size_t aria_paged_workspace_counter_bytes(void) {
  const size_t a = paged_counter_bytes(), b = prompt_counter_bytes();
  return a > b ? a : b;
}

int aria_stream_capture_id(void* stream, unsigned long long* id) {
  if (!id) return ARIA_Q4_EINVAL;
  *id = 0;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long of = 0;
  if (cudaError_t e = cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &of)) return cuda_status(e);
  if (status == cudaStreamCaptureStatusActive) *id = of;
  return ARIA_Q4_OK;
}

size_t aria_attention_paged_workspace_bytes(const aria_paged_kv* kv, int M, int heads, int weights) {
  long long slots = 0;
  if (check_kv(kv, M, &slots) != ARIA_Q4_OK || heads <= 0 || heads % kv->kv_heads) return 0;
  return paged_workspace_bytes(M, heads, kv->kv_heads, kv->head_dim, slots, weights != 0);
}

int aria_attention_paged(const aria_paged_kv* kv, int M, int heads, const uint16_t* q, long long q_row,
                         long long q_head, const uint16_t* k_new, const uint16_t* v_new, long long new_row,
                         long long new_head, float scale, uint16_t* out, long long out_row, long long out_head,
                         float* lse, const float* weights_in, float* weights_out, long long weights_cap,
                         int* slot_pos, const int* positions, void* workspace, size_t workspace_bytes, void* stream) {
  long long slots = 0;
  if (int s = check_kv(kv, M, &slots)) return s;
  if (heads <= 0 || heads % kv->kv_heads || !(scale == scale)) return ARIA_Q4_EINVAL;
  // tiles of 16 slots of all pairs (sequence, head), counted in 31 bits
  if ((long long)M * ((slots + 15) / 16) > 0x7fffffffLL / heads) return ARIA_Q4_ESIZE;
  if ((k_new == nullptr) != (v_new == nullptr) || (weights_in == nullptr) != (weights_out == nullptr))
    return ARIA_Q4_EINVAL;
  if (slot_pos && (!weights_out || !k_new || !positions)) return ARIA_Q4_EINVAL;
  if (weights_out && weights_cap < slots) return ARIA_Q4_ESIZE;
  if (M == 0) return ARIA_Q4_OK;
  if (!q || !out || !workspace) return ARIA_Q4_EINVAL;
  if (!aligned16(q) || q_row % 8 || q_head % 8) return ARIA_Q4_EALIGN;
  if (!elements_aligned(2, {out}) || !elements_aligned(4, {lse, weights_in, weights_out, slot_pos, positions}))
    return ARIA_Q4_EALIGN;
  if (k_new && (!aligned16(k_new) || !aligned16(v_new) || new_row % 8 || new_head % 8)) return ARIA_Q4_EALIGN;
  if (((uintptr_t)workspace & 255u) != 0) return ARIA_Q4_EALIGN;
  if (int s = check_device()) return s;
  if (workspace_bytes < paged_workspace_bytes(M, heads, kv->kv_heads, kv->head_dim, slots, weights_out != nullptr))
    return ARIA_Q4_ESIZE;
  PagedArgs a = {};
  a.M = M;
  a.Hq = heads;
  a.Hkv = kv->kv_heads;
  a.G = heads / kv->kv_heads;
  a.q = q;
  a.q_row = q_row;
  a.q_head = q_head;
  a.k_pages = a.k_pages_w = (uint16_t*)kv->k_pages;
  a.v_pages = a.v_pages_w = (uint16_t*)kv->v_pages;
  a.page_stride = kv->page_stride;
  a.slot_stride = kv->slot_stride;
  a.head_stride = kv->head_stride;
  a.num_pages = kv->num_pages;
  a.page_size = kv->page_size;
  a.table = kv->block_table;
  a.table_stride = kv->table_stride;
  a.max_pages = kv->max_pages;
  a.lens = kv->lens;
  a.k_new = k_new;
  a.v_new = v_new;
  a.new_row = new_row;
  a.new_head = new_head;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  a.out_row = out_row;
  a.out_head = out_head;
  a.lse = lse;
  a.slots = slots;
  return cuda_status(launch_attention_paged(a, kv->head_dim, kv->dtype == ARIA_Q4_BF16, workspace, weights_in,
                                            weights_out, weights_cap, slot_pos, positions, (cudaStream_t)stream));
}

size_t aria_prompt_weights_workspace_bytes(int B, int T, int heads, int kv_heads, int first_query) {
  if (B <= 0 || T <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || first_query < 0 ||
      !prompt_blocks_fit(B, T, heads, kv_heads))
    return 0;
  return prompt_workspace_bytes(B, T, kv_heads, heads / kv_heads, first_query);
}

int aria_prompt_weights(const uint16_t* q, long long q_seq, long long q_pos, long long q_head, const uint16_t* k,
                        long long k_seq, long long k_pos, long long k_head, int dtype, int B, int T, int heads,
                        int kv_heads, int head_dim, const float* lse, float scale, int first_query, float* weights,
                        long long w_seq, long long w_head, void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || T < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || first_query < 0 || !(scale == scale))
    return ARIA_Q4_EINVAL;
  if (dtype != ARIA_Q4_F16 && dtype != ARIA_Q4_BF16) return ARIA_Q4_EINVAL;
  if (head_dim != 64 && head_dim != 128) return ARIA_Q4_EUNSUPPORTED;
  if (B == 0 || T == 0) return ARIA_Q4_OK;
  if (!q || !k || !lse || !weights) return ARIA_Q4_EINVAL;
  if (!aligned16(q) || !aligned16(k) || !elements_aligned(4, {lse, weights})) return ARIA_Q4_EALIGN;
  const long long strides[6] = {q_seq, q_pos, q_head, k_seq, k_pos, k_head};
  for (long long s : strides) {
    if (s <= 0) return ARIA_Q4_EINVAL;
    if (s % 8) return ARIA_Q4_EALIGN;
    if (s >= (1LL << 38)) return ARIA_Q4_ESIZE;  // the tensor maps' strides are 40 bits of bytes
  }
  if (!prompt_blocks_fit(B, T, heads, kv_heads)) return ARIA_Q4_ESIZE;
  if (((uintptr_t)workspace & 255u) != 0) return ARIA_Q4_EALIGN;
  if (int s = check_device()) return s;
  const size_t need = prompt_workspace_bytes(B, T, kv_heads, heads / kv_heads, first_query);
  if (need > 0 && !workspace) return ARIA_Q4_EINVAL;
  if (workspace_bytes < need) return ARIA_Q4_ESIZE;
  return cuda_status(launch_prompt_weights(q, k, dtype == ARIA_Q4_BF16, head_dim, q_seq, q_pos, q_head, k_seq, k_pos,
                                           k_head, B, T, kv_heads, heads / kv_heads, first_query, scale, lse, weights,
                                           w_seq, w_head, workspace, (cudaStream_t)stream));
}

size_t aria_cache_evict_workspace_bytes(const aria_paged_kv* kv, int M, int keep) {
  long long slots = 0;
  if (check_kv(kv, M, &slots) != ARIA_Q4_OK || keep <= 0) return 0;
  return evict_workspace_bytes(M, kv->kv_heads, slots, keep);
}

int aria_cache_evict(const aria_paged_kv* kv, int M, const float* weights_in, float* weights_out, const int* pos_in,
                     int* pos_out, long long cap, const int* next_pos, int keep, int recent, int sinks, int* lens_out,
                     void* workspace, size_t workspace_bytes, void* stream) {
  long long slots = 0;
  if (int s = check_kv(kv, M, &slots)) return s;
  if (keep <= 0 || recent < 0 || sinks < 0 || (long long)recent + sinks > keep) return ARIA_Q4_EINVAL;
  if (cap < slots || slots > kEvictMaxSlots) return ARIA_Q4_ESIZE;
  if (M == 0) return ARIA_Q4_OK;
  if (!weights_in || !weights_out || !pos_in || !pos_out || !next_pos || lens_out == kv->lens) return ARIA_Q4_EINVAL;
  if (!elements_aligned(4, {weights_in, weights_out, pos_in, pos_out, next_pos, lens_out})) return ARIA_Q4_EALIGN;
  if ((long long)M * kv->kv_heads > 0x7fffffffLL / 8) return ARIA_Q4_ESIZE;
  const size_t need = evict_workspace_bytes(M, kv->kv_heads, slots, keep);
  if (need > 0 && !workspace) return ARIA_Q4_EINVAL;
  if (workspace_bytes < need) return ARIA_Q4_ESIZE;
  if (((uintptr_t)workspace & 255u) != 0) return ARIA_Q4_EALIGN;
  if (int s = check_device()) return s;
  EvictArgs a = {};
  a.M = M;
  a.Hkv = kv->kv_heads;
  a.k_pages = (uint16_t*)kv->k_pages;
  a.v_pages = (uint16_t*)kv->v_pages;
  a.page_stride = kv->page_stride;
  a.slot_stride = kv->slot_stride;
  a.head_stride = kv->head_stride;
  a.num_pages = kv->num_pages;
  a.page_size = kv->page_size;
  a.table = kv->block_table;
  a.table_stride = kv->table_stride;
  a.max_pages = kv->max_pages;
  a.lens = kv->lens;
  a.slots = slots;
  a.weights_in = weights_in;
  a.weights_out = weights_out;
  a.pos_in = pos_in;
  a.pos_out = pos_out;
  a.cap = cap;
  a.next_pos = next_pos;
  a.lens_out = lens_out;
  a.keep = keep;
  a.recent = recent;
  a.sinks = sinks;
  a.row_bytes = kv->head_dim * 2;
  return cuda_status(launch_cache_evict(a, workspace, (cudaStream_t)stream));
}

size_t aria_logits_workspace_bytes(int M) { return M > 0 ? logits_workspace_bytes(M) : 0; }

int aria_logits_adjust(const aria_logit_rules* r, const void* logits, int dtype, long long logits_row, int M, int V,
                       void* out, int out_dtype, long long out_row, int* token, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (!r || M < 0 || V <= 0 || M > 65535) return ARIA_Q4_EINVAL;
  if (dtype != ARIA_Q4_F32 && dtype != ARIA_Q4_F16 && dtype != ARIA_Q4_BF16) return ARIA_Q4_EINVAL;
  if (out_dtype != dtype && out_dtype != ARIA_Q4_F32) return ARIA_Q4_EINVAL;
  if (r->history && (!r->history_lens || r->history_cap < 0)) return ARIA_Q4_EINVAL;
  if (r->bias_tokens && (!r->bias_values || r->biases < 0)) return ARIA_Q4_EINVAL;
  if (r->allowed_row < 0 || logits_row < 0 || out_row < 0) return ARIA_Q4_EINVAL;
  // indexes run in 31 bits, up to a chunk and a block's step past the last one
  const int most = 0x7fffffff - (1 << 16);
  if (V > most || r->history_cap > most || r->biases > most) return ARIA_Q4_ESIZE;
  if (M == 0) return ARIA_Q4_OK;
  if (!logits || !out) return ARIA_Q4_EINVAL;
  if (!elements_aligned(dtype == ARIA_Q4_F32 ? 4 : 2, {logits}) ||
      !elements_aligned(out_dtype == ARIA_Q4_F32 ? 4 : 2, {out}) ||
      !elements_aligned(4, {r->history, r->history_lens, r->prompt_lens, r->repetition, r->frequency, r->presence,
                            r->bias_tokens, r->bias_values, r->allowed, token}))
    return ARIA_Q4_EALIGN;
  if (out == logits && (out_dtype != dtype || out_row != logits_row)) return ARIA_Q4_EINVAL;
  if (token) {
    if (!workspace) return ARIA_Q4_EINVAL;
    if (workspace_bytes < logits_workspace_bytes(M)) return ARIA_Q4_ESIZE;
    if (((uintptr_t)workspace & 255u) != 0) return ARIA_Q4_EALIGN;
  }
  if (int s = check_device()) return s;
  LogitArgs a = {};
  a.M = M;
  a.V = V;
  a.logits = logits;
  a.logits_row = logits_row;
  a.out = out;
  a.out_row = out_row;
  a.history = r->history;
  a.history_row = r->history_row;
  a.history_cap = r->history_cap;
  a.history_lens = r->history_lens;
  a.prompt_lens = r->prompt_lens;
  a.repetition = r->repetition;
  a.frequency = r->frequency;
  a.presence = r->presence;
  if (r->bias_tokens && r->biases > 0) {  // without the list its length says nothing
    a.bias_tokens = r->bias_tokens;
    a.bias_values = r->bias_values;
    a.bias_row = r->bias_row;
    a.biases = r->biases;
  }
  a.allowed = r->allowed;
  a.allowed_row = r->allowed_row;
  a.token = token;
  auto code = [](int d) { return d == ARIA_Q4_BF16 ? 2 : d; };
  return cuda_status(launch_logits_adjust(a, code(dtype), code(out_dtype), token ? workspace : nullptr,
                                          (cudaStream_t)stream));
}

}  // extern "C"
