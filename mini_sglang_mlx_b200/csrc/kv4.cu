// C-ABI entry points of the 4-bit K/V pool: rows in and out, norm + rotation + append, decode and prefill attention.
// Declarations: include/msgl_b200.h.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "decode_q4.cuh"
#include "host_common.cuh"
#include "kv4_project.cuh"
#include "prefill_tc.cuh"

using namespace msgl_host;

namespace {

// What every operator over the pool asks of it.
int check_pool(const char* op, int num_kv_heads, int head_dim, int64_t num_slots, int dtype) {
  if (num_kv_heads <= 0 || num_slots < 0)
    return fail(MSGL_BAD_SHAPE, std::string(op) + "the pools must be (num_blocks, num_kv_heads, 9 * head_dim / 2)");
  if (head_dim != 128 && head_dim != 256)
    return fail(MSGL_UNSUPPORTED_HEAD_DIM, std::string(op) + "head_dim must be 128 or 256");
  if (dtype != MSGL_DTYPE_BF16 && dtype != MSGL_DTYPE_F16)
    return fail(MSGL_BAD_DTYPE, std::string(op) + "unsupported dtype, must be float16 or bfloat16");
  if (num_slots % msgl::kKv4Rows != 0 || num_slots >= (1ll << 31))
    return fail(MSGL_BAD_SHAPE, std::string(op) + "num_slots must be a multiple of 16 below 2^31");
  if (num_kv_heads > 65535) return fail(MSGL_BAD_SHAPE, std::string(op) + "num_kv_heads must be <= 65535");
  return MSGL_OK;
}

unsigned grid_of(int64_t threads, int per_sm) {
  int sms = sm_count_cached();
  if (sms <= 0) sms = 148;
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, static_cast<int64_t>(sms) * per_sm)));
}

// ---- decode scheduling, in blocks of 16 tokens
constexpr int kQ4MinShare = 8;
constexpr int kQ4MaxShare = 1024;
constexpr int kQ4Pad = 12;

struct Q4Plan {
  int col_tiles, cols;       // CTAs side by side, columns of each
  int64_t shares;
  size_t ticket_bytes, part_bytes;
};
// `columns` of a sequence at most, `blocks` of all sequences at most.
Q4Plan plan_q4(int batch, int columns, int hkv, int head_dim, int64_t blocks, int sms) {
  Q4Plan pl{};
  pl.cols = head_dim == 128 && columns > 8 ? 16 : 8;
  pl.col_tiles = (columns + pl.cols - 1) / pl.cols;
  constexpr int ctas_per_sm = 1;
  const int64_t wave = std::max(1, sms * ctas_per_sm / (hkv * pl.col_tiles));
  blocks += static_cast<int64_t>(batch) * kQ4Pad;
  pl.shares = wave * std::max<int64_t>(1, (blocks + wave * kQ4MaxShare - 1) / (wave * kQ4MaxShare));
  const size_t tickets = static_cast<size_t>(batch) * hkv * pl.col_tiles;
  pl.ticket_bytes = tickets <= kTicketSlots ? 0 : (tickets * sizeof(int) + 255) / 256 * 256;
  pl.part_bytes = static_cast<size_t>(pl.shares) * 2 * hkv * pl.col_tiles * pl.cols * msgl::q4_partial_floats(head_dim) * sizeof(float);
  return pl;
}

template <typename T, int HD, int NT, bool BLOCKS, int U, int WARPS, int STAGES, int MINB>
cudaError_t launch_q4(const msgl::Q4DecodeParams& p, cudaStream_t s) {
  auto* kernel = msgl::q4_decode_kernel<T, HD, NT, BLOCKS, U, WARPS, STAGES, MINB>;
  constexpr int smem = msgl::q4_decode_smem(HD, WARPS, STAGES * U);
  const cudaError_t e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(p.num_shares * p.col_tiles * p.hkv)), dim3(WARPS * 32), smem, s, p);
}
template <bool BLOCKS>
cudaError_t launch_q4_any(const msgl::Q4DecodeParams& p, int head_dim, int cols, int dtype, cudaStream_t s) {
  auto go = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    if (head_dim == 256) return launch_q4<T, 256, 1, BLOCKS, 1, 12, 3, 1>(p, s);
    return cols == 8 ? launch_q4<T, 128, 1, BLOCKS, 2, 12, 3, 1>(p, s) : launch_q4<T, 128, 2, BLOCKS, 1, 12, 6, 1>(p, s);
  };
  return dtype == MSGL_DTYPE_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

// The rest of a call's parameters, and its launch.
template <bool BLOCKS>
int run_q4(const char* op, msgl::Q4DecodeParams& p, const Q4Plan& pl, void* workspace, size_t workspace_bytes, int head_dim,
           int dtype, void* stream) {
  if (!workspace || workspace_bytes < kStatusBytes + pl.ticket_bytes + pl.part_bytes)
    return fail(MSGL_BAD_ARG, std::string(op) + ": workspace too small");
  if (pl.shares * pl.col_tiles * p.hkv > 0x7fffffffLL)
    return fail(MSGL_BAD_SHAPE, std::string(op) + ": problem too large for one launch");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.status = reinterpret_cast<int*>(ws);
  p.tickets = reinterpret_cast<int*>(ws + (pl.ticket_bytes == 0 ? 256 : kStatusBytes));
  p.part = reinterpret_cast<float*>(ws + kStatusBytes + pl.ticket_bytes);
  if (pl.ticket_bytes != 0) {
    const cudaError_t e = cudaMemsetAsync(p.tickets, 0, pl.ticket_bytes, s);
    if (e != cudaSuccess) return cuda_fail(op, e);
  }
  p.col_tiles = pl.col_tiles;
  p.num_shares = static_cast<int>(pl.shares);
  p.min_share = kQ4MinShare;
  p.pad = kQ4Pad;
  const cudaError_t e = launch_q4_any<BLOCKS>(p, head_dim, pl.cols, dtype, s);
  return e == cudaSuccess ? MSGL_OK : cuda_fail(op, e);
}

// Query blocks of few columns per KV head run the decode kernel (decode_q4.cuh), others the one-CTA tcgen05 kernel.
constexpr int kQ4BlockColumns = 16;
bool q4_block_form(int max_len_extend, int group) {
  return static_cast<int64_t>(max_len_extend) * group <= kQ4BlockColumns;
}
// Blocks of a call at most: what the pages hold, or what a window leaves.
int64_t q4_block_bound(int batch, int64_t total_pages, int page_size, int max_len_extend, int window) {
  const int64_t all = total_pages * page_size / msgl::kKv4Rows;
  return window > 0 ? std::min<int64_t>(all, batch * ((static_cast<int64_t>(window) + max_len_extend) / msgl::kKv4Rows + 2)) : all;
}

}  // namespace

extern "C" {

int msgl_store_kv_cache_q4(void* k_cache, void* v_cache, const int32_t* indices, const void* k, const void* v, int length,
                           int num_kv_heads, int head_dim, int64_t num_slots, int64_t k_token_stride,
                           int64_t v_token_stride, int dtype, void* status_word, void* stream) {
  const char* op = "store_kv_cache_q4: ";
  if (length < 0) return fail(MSGL_BAD_SHAPE, std::string(op) + "k and v shape must be (length, num_kv_heads, head_dim)");
  if (const int rc = check_pool(op, num_kv_heads, head_dim, num_slots, dtype)) return rc;
  const int64_t row = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (length > 1 && (k_token_stride < row || v_token_stride < row))
    return fail(MSGL_BAD_SHAPE, std::string(op) + "row stride smaller than num_kv_heads*head_dim");
  if (length == 0) return MSGL_OK;
  if (!k_cache || !v_cache || !indices || !k || !v) return fail(MSGL_BAD_ARG, std::string(op) + "null tensor pointer");
  auto aligned = [](const void* ptr, int a) { return reinterpret_cast<uintptr_t>(ptr) % a == 0; };
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned(k, 8) || !aligned(v, 8) || k_token_stride % 4 != 0 ||
      v_token_stride % 4 != 0)
    return fail(MSGL_BAD_ARG, std::string(op) + "k and v rows must be 8-byte aligned, the pools 16-byte aligned");
  msgl::Kv4StoreParams p{};
  p.k_pool = static_cast<unsigned char*>(k_cache);
  p.v_pool = static_cast<unsigned char*>(v_cache);
  p.k = k;
  p.v = v;
  p.slots = indices;
  p.k_stride = k_token_stride;
  p.v_stride = v_token_stride;
  p.num_slots = num_slots;
  p.n = length;
  p.hkv = num_kv_heads;
  p.wide = aligned16(k) && aligned16(v) && k_token_stride % 8 == 0 && v_token_stride % 8 == 0;
  p.status = static_cast<int*>(status_word);
  auto* kernel = head_dim == 256 ? (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_store_kernel<__nv_bfloat16, 256>
                                                             : msgl::kv4_store_kernel<__half, 256>)
                                 : (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_store_kernel<__nv_bfloat16, 128>
                                                             : msgl::kv4_store_kernel<__half, 128>);
  const cudaError_t e = launch_dependent(kernel, dim3(grid_of(length * row / 8, 16)), dim3(256), 0,
                                         static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? MSGL_OK : cuda_fail("store_kv_cache_q4", e);
}

int msgl_load_kv_cache_q4(const void* k_cache, const void* v_cache, const int32_t* indices, void* k, void* v, int length,
                          int num_kv_heads, int head_dim, int64_t num_slots, int dtype, void* status_word, void* stream) {
  const char* op = "load_kv_cache_q4: ";
  if (length < 0) return fail(MSGL_BAD_SHAPE, std::string(op) + "negative length");
  if (const int rc = check_pool(op, num_kv_heads, head_dim, num_slots, dtype)) return rc;
  if (length == 0) return MSGL_OK;
  if (!k_cache || !v_cache || !indices || !k || !v) return fail(MSGL_BAD_ARG, std::string(op) + "null tensor pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k) || !aligned16(v))
    return fail(MSGL_BAD_ARG, std::string(op) + "k, v and the pools must be 16-byte aligned");
  msgl::Kv4LoadParams p{};
  p.k_pool = static_cast<const unsigned char*>(k_cache);
  p.v_pool = static_cast<const unsigned char*>(v_cache);
  p.k = k;
  p.v = v;
  p.slots = indices;
  p.num_slots = num_slots;
  p.n = length;
  p.hkv = num_kv_heads;
  p.status = static_cast<int*>(status_word);
  auto* kernel = head_dim == 256 ? (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_load_kernel<__nv_bfloat16, 256>
                                                             : msgl::kv4_load_kernel<__half, 256>)
                                 : (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_load_kernel<__nv_bfloat16, 128>
                                                             : msgl::kv4_load_kernel<__half, 128>);
  const cudaError_t e = launch_dependent(kernel, dim3(grid_of(static_cast<int64_t>(length) * num_kv_heads * head_dim / 8, 16)),
                                         dim3(256), 0, static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? MSGL_OK : cuda_fail("load_kv_cache_q4", e);
}

int msgl_qk_norm_rope_store_q4(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                               const int32_t* positions, const int32_t* out_loc, void* q_out, void* k_cache, void* v_cache,
                               int n_tokens, int num_q_heads, int num_kv_heads, int head_dim, int rotary_dim, double rope_base,
                               float eps, int64_t num_slots, int64_t q_token_stride, int64_t k_token_stride,
                               int64_t v_token_stride, int dtype, void* status_word, void* stream) {
  const char* op = "qk_norm_rope_store_q4: ";
  if (n_tokens < 0 || num_q_heads <= 0)
    return fail(MSGL_BAD_SHAPE, std::string(op) +
                "q must be (n_tokens, num_q_heads, head_dim), k and v (n_tokens, num_kv_heads, head_dim)");
  if (const int rc = check_pool(op, num_kv_heads, head_dim, num_slots, dtype)) return rc;
  if (rotary_dim != head_dim && rotary_dim != head_dim / 2 && rotary_dim != head_dim / 4)
    return fail(MSGL_BAD_ARG, std::string(op) + "rotary_dim must be head_dim, head_dim/2 or head_dim/4");
  if (!(rope_base > 1.) || !(eps >= 0.f))
    return fail(MSGL_BAD_ARG, std::string(op) + "rope_base must be > 1 and eps >= 0");
  const int64_t kv_row = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (n_tokens > 1 && (q_token_stride < static_cast<int64_t>(num_q_heads) * head_dim || k_token_stride < kv_row ||
                       v_token_stride < kv_row))
    return fail(MSGL_BAD_SHAPE, std::string(op) + "a token stride is smaller than its row");
  if (n_tokens == 0) return MSGL_OK;
  if (!q || !k || !v || !positions || !out_loc || !q_out || !k_cache || !v_cache)
    return fail(MSGL_BAD_ARG, std::string(op) + "null tensor pointer");
  auto aligned = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 8 == 0; };
  if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(q_weight) || !aligned(k_weight) || q_token_stride % 4 != 0 ||
      k_token_stride % 4 != 0 || v_token_stride % 4 != 0 || !aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache))
    return fail(MSGL_BAD_ARG, std::string(op) + "q, k and v rows and the norm weights must be 8-byte aligned, the pools and "
                                                "the result 16-byte aligned");
  constexpr int R = msgl::kKv4RowsPerItem;
  const int64_t items = static_cast<int64_t>(n_tokens) * ((num_q_heads + R - 1) / R + 2 * ((num_kv_heads + R - 1) / R));
  if (items >= (1ll << 31)) return fail(MSGL_BAD_ARG, std::string(op) + "too many rows for one call");
  msgl::Kv4ProjectParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.positions = positions;
  p.slots = out_loc;
  p.k_pool = static_cast<unsigned char*>(k_cache);
  p.v_pool = static_cast<unsigned char*>(v_cache);
  p.n = n_tokens;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.rotary_dim = rotary_dim;
  p.q_stride = q_token_stride;
  p.k_stride = k_token_stride;
  p.v_stride = v_token_stride;
  p.num_slots = num_slots;
  p.log2_base = std::log2(rope_base);
  p.eps = eps;
  p.status = static_cast<int*>(status_word);
  auto* kernel = head_dim == 256 ? (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_project_kernel<__nv_bfloat16, 256>
                                                             : msgl::kv4_project_kernel<__half, 256>)
                                 : (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_project_kernel<__nv_bfloat16, 128>
                                                             : msgl::kv4_project_kernel<__half, 128>);
  const cudaError_t e = launch_dependent(kernel, dim3(grid_of(items * msgl::kv4_project_lanes(head_dim), 16)), dim3(256), 0,
                                         static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? MSGL_OK : cuda_fail("qk_norm_rope_store_q4", e);
}

size_t msgl_decode_workspace_bytes_q4(int batch, int num_q_heads, int num_kv_heads, int head_dim, int64_t total_pages,
                                      int page_size) {
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || total_pages < 0 || page_size <= 0)
    return kStatusBytes;
  const int sms = sm_count_cached();
  const Q4Plan pl = plan_q4(batch, std::max(1, num_q_heads / num_kv_heads), num_kv_heads, head_dim,
                            total_pages * page_size / msgl::kKv4Rows, sms > 0 ? sms : 148);
  return kStatusBytes + pl.ticket_bytes + pl.part_bytes;
}

int msgl_paged_decode_attention_q4(const void* q, const void* k_cache, const void* v_cache, const int32_t* page_indptr,
                                   const int32_t* page_indices, const int32_t* kv_lens, const void* gate, void* out,
                                   void* workspace, size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads,
                                   int head_dim, int64_t num_slots, int dtype, float sm_scale, int page_size,
                                   int64_t total_pages, void* stream) {
  const char* op = "paged_decode_attention_q4: ";
  if (batch < 0 || num_q_heads <= 0)
    return fail(MSGL_BAD_SHAPE, std::string(op) + "q must be 3D (batch, num_q_heads, head_dim)");
  if (const int rc = check_pool(op, num_kv_heads, head_dim, num_slots, dtype)) return rc;
  if (num_q_heads % num_kv_heads != 0)
    return fail(MSGL_BAD_GQA, std::string(op) + "num_q_heads must be a multiple of num_kv_heads");
  if (num_q_heads / num_kv_heads > 16)
    return fail(MSGL_BAD_GQA, std::string(op) + "only q_heads/kv_heads <= 16 is supported");
  if (page_size <= 0 || page_size % msgl::kKv4Rows != 0)
    return fail(MSGL_BAD_ARG, std::string(op) + "page_size must be a multiple of 16");
  if (total_pages < 0 || total_pages >= (1ll << 31) / page_size)
    return fail(MSGL_BAD_SHAPE, std::string(op) + "fewer than 2^31 tokens in all pages");
  if (batch == 0) return MSGL_OK;
  if (batch > 65535) return fail(MSGL_BAD_SHAPE, std::string(op) + "batch must be <= 65535");
  if (!q || !k_cache || !v_cache || !out || !page_indptr || !kv_lens || (total_pages > 0 && !page_indices))
    return fail(MSGL_BAD_ARG, std::string(op) + "null tensor pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || !aligned16(gate) ||
      !aligned16(workspace))
    return fail(MSGL_BAD_ARG, std::string(op) + "q, the pools, out, gate and the workspace must be 16-byte aligned");
  const int sms = sm_count_cached();
  if (sms <= 0) return fail(MSGL_CUDA_ERROR, std::string(op) + "cannot query the device");
  const Q4Plan pl = plan_q4(batch, num_q_heads / num_kv_heads, num_kv_heads, head_dim,
                            total_pages * page_size / msgl::kKv4Rows, sms);
  msgl::Q4DecodeParams p{};
  p.q = q;
  p.k_pool = static_cast<const unsigned char*>(k_cache);
  p.v_pool = static_cast<const unsigned char*>(v_cache);
  p.page_indptr = page_indptr;
  p.page_indices = page_indices;
  p.kv_lens = kv_lens;
  p.page_blocks = page_size / msgl::kKv4Rows;
  p.total_pages = static_cast<int>(total_pages);
  p.out = out;
  p.gate = gate;
  p.batch = batch;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.num_blocks = num_slots / msgl::kKv4Rows;
  p.scale_log2 = sm_scale * msgl::kLog2e;
  return run_q4<false>("paged_decode_attention_q4", p, pl, workspace, workspace_bytes, head_dim, dtype, stream);
}

size_t msgl_prefill_workspace_bytes_q4(int batch, int total_q, int64_t total_pages, int page_size, int num_q_heads,
                                       int num_kv_heads, int head_dim, int max_len_extend, int sliding_window_size) {
  if (batch <= 0 || total_q <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || total_pages < 0 || page_size <= 0)
    return kStatusBytes;
  max_len_extend = std::max(1, max_len_extend);
  const int group = std::max(1, num_q_heads / num_kv_heads);
  if (!q4_block_form(max_len_extend, group))
    return msgl_prefill_workspace_bytes(batch, total_q, total_pages * page_size, num_q_heads, num_kv_heads, head_dim,
                                        max_len_extend, sliding_window_size);
  const int sms = sm_count_cached();
  const Q4Plan pl = plan_q4(batch, max_len_extend * group, num_kv_heads, head_dim,
                            q4_block_bound(batch, total_pages, page_size, max_len_extend, sliding_window_size), sms > 0 ? sms : 148);
  return kStatusBytes + pl.ticket_bytes + pl.part_bytes;
}

int msgl_paged_prefill_attention_q4(const void* q, const void* k_cache, const void* v_cache, const int32_t* qo_indptr,
                                    const int32_t* page_indptr, const int32_t* page_indices, const int32_t* kv_lens,
                                    const int32_t* prefix_lens, const void* gate, void* out, void* workspace,
                                    size_t workspace_bytes, int batch, int total_q, int num_q_heads, int num_kv_heads,
                                    int head_dim, int64_t num_slots, int dtype, float sm_scale, int max_len_extend,
                                    int is_cross_attention, int sliding_window_size, int page_size, int64_t total_pages,
                                    void* stream) {
  const char* op = "paged_prefill_attention_q4: ";
  if (total_q < 0 || num_q_heads <= 0)
    return fail(MSGL_BAD_SHAPE, std::string(op) + "q must be 3D (total_q_tokens, num_q_heads, head_dim)");
  if (const int rc = check_pool(op, num_kv_heads, head_dim, num_slots, dtype)) return rc;
  if (num_q_heads % num_kv_heads != 0)
    return fail(MSGL_BAD_GQA, std::string(op) + "num_q_heads must be a multiple of num_kv_heads");
  if (num_q_heads > 65535) return fail(MSGL_BAD_SHAPE, std::string(op) + "num_q_heads must be <= 65535");
  if (sliding_window_size < 0) return fail(MSGL_BAD_ARG, std::string(op) + "sliding_window_size must be >= 0");
  if (batch <= 0) return fail(MSGL_BAD_SHAPE, std::string(op) + "batch must be > 0");
  if (page_size <= 0 || page_size % msgl::kKv4Rows != 0)
    return fail(MSGL_BAD_ARG, std::string(op) + "page_size must be a multiple of 16");
  if (total_pages < 0 || total_pages >= (1ll << 31) / page_size)
    return fail(MSGL_BAD_SHAPE, std::string(op) + "fewer than 2^31 tokens in all pages");
  if (total_q == 0) return MSGL_OK;
  if (max_len_extend < 1) max_len_extend = 1;
  if (!q || !k_cache || !v_cache || !qo_indptr || !page_indptr || !kv_lens || !prefix_lens || !out ||
      (total_pages > 0 && !page_indices))
    return fail(MSGL_BAD_ARG, std::string(op) + "null tensor pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || !aligned16(gate) ||
      !aligned16(workspace))
    return fail(MSGL_BAD_ARG, std::string(op) + "q, the pools, out, gate and the workspace must be 16-byte aligned");
  const int sms = sm_count_cached();
  if (sms <= 0) return fail(MSGL_CUDA_ERROR, std::string(op) + "cannot query the device");
  if (batch <= 65535 && q4_block_form(max_len_extend, num_q_heads / num_kv_heads)) {
    const Q4Plan blocks = plan_q4(batch, max_len_extend * (num_q_heads / num_kv_heads), num_kv_heads, head_dim,
                                  q4_block_bound(batch, total_pages, page_size, max_len_extend, sliding_window_size), sms);
    msgl::Q4DecodeParams p{};
    p.q = q;
    p.k_pool = static_cast<const unsigned char*>(k_cache);
    p.v_pool = static_cast<const unsigned char*>(v_cache);
    p.page_indptr = page_indptr;
    p.page_indices = page_indices;
    p.kv_lens = kv_lens;
    p.qo_indptr = qo_indptr;
    p.prefix_lens = prefix_lens;
    p.page_blocks = page_size / msgl::kKv4Rows;
    p.total_pages = static_cast<int>(total_pages);
    p.out = out;
    p.gate = gate;
    p.batch = batch;
    p.hq = num_q_heads;
    p.hkv = num_kv_heads;
    p.group = num_q_heads / num_kv_heads;
    p.is_cross = is_cross_attention ? 1 : 0;
    p.window = sliding_window_size;
    p.num_blocks = num_slots / msgl::kKv4Rows;
    p.scale_log2 = sm_scale * msgl::kLog2e;
    return run_q4<true>("paged_prefill_attention_q4", p, blocks, workspace, workspace_bytes, head_dim, dtype, stream);
  }
  const PrefillPlan pl = plan_prefill(batch, total_q, total_pages * page_size, num_q_heads, num_kv_heads, head_dim,
                                      max_len_extend, sliding_window_size, sms);
  if (!workspace || workspace_bytes < kStatusBytes + pl.plan_bytes + pl.part_ml_bytes + pl.part_o_bytes)
    return fail(MSGL_BAD_ARG, std::string(op) + "workspace too small");
  if (pl.items * num_kv_heads > 0x7fffffffLL)
    return fail(MSGL_BAD_SHAPE, std::string(op) + "problem too large for one launch");
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  msgl::PrefillParams p{};
  p.q = q;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.qo_indptr = qo_indptr;
  p.prefix_lens = prefix_lens;
  p.page_indptr = page_indptr;
  p.page_indices = page_indices;
  p.kv_lens = kv_lens;
  p.page_size = page_size;
  p.out = out;
  p.gate = gate;
  p.status = reinterpret_cast<int*>(ws);
  if (pl.kv_chunk > 0) {
    p.tickets = pl.fused_merge ? reinterpret_cast<int*>(ws + 256) : nullptr;
    p.part_ml = reinterpret_cast<float*>(ws + kStatusBytes + pl.plan_bytes);
    p.part_o = reinterpret_cast<float*>(ws + kStatusBytes + pl.plan_bytes + pl.part_ml_bytes);
  }
  p.batch = batch;
  p.total_q = total_q;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.num_slots = num_slots;
  p.scale_log2 = sm_scale * msgl::kLog2e;
  p.is_cross = is_cross_attention ? 1 : 0;
  p.window = sliding_window_size;
  p.kv_chunk = pl.kv_chunk;
  p.group_recip = msgl::reciprocal(p.group);
  p.page_recip = msgl::reciprocal(page_size);
  p.chunk_recip = msgl::reciprocal(p.kv_chunk);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CUtensorMap none, tm_q;
  std::memset(&none, 0, sizeof(none));
  std::memset(&tm_q, 0, sizeof(tm_q));
  p.q_tma = make_query_tensor_map(&tm_q, q, total_q, num_q_heads, p.group, head_dim, dtype) ? 1 : 0;
  const dim3 grid(static_cast<unsigned>(pl.items * num_kv_heads));
  auto launch = [&](auto kernel, auto merge, int threads, int smem) -> cudaError_t {
    cudaError_t err = allow_smem(kernel, smem);
    if (err != cudaSuccess) return err;
    err = launch_dependent(kernel, grid, dim3(threads), smem, s, p, none, none, tm_q);
    if (err != cudaSuccess) return err;
    if (pl.kv_chunk > 0 && !pl.fused_merge)
      return launch_dependent(merge, dim3(grid.x, msgl::kMergeSlices), dim3(msgl::kMergeWarps * 32), 0, s, p);
    return cudaSuccess;
  };
  auto dispatch = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    using S1 = msgl::TcShape<1>;
    using S2 = msgl::TcShape<2>;
    using S1w = msgl::TcShape<1, 256>;
    if (head_dim == 256)
      return launch(msgl::prefill_tc_kernel<T, 64, 1, 256, false, true>, msgl::prefill_merge_kernel<T, 256, S1w::kBM>,
                    S1w::kThreads, msgl::Kv4Shape<1, 256>::kSmemBytes);
    if (prefill_short_q(max_len_extend, p.group, head_dim))
      return launch(msgl::prefill_tc_kernel<T, 64, 1, 128, false, true>, msgl::prefill_merge_kernel<T, 128, S1::kBM>,
                    S1::kThreads, msgl::Kv4Shape<1, 128>::kSmemBytes);
    return launch(msgl::prefill_tc_kernel<T, 128, 2, 128, false, true>, msgl::prefill_merge_kernel<T, 128, S2::kBM>,
                  S2::kThreads, msgl::Kv4Shape<2, 128>::kSmemBytes);
  };
  const cudaError_t e = dtype == MSGL_DTYPE_BF16 ? dispatch(__nv_bfloat16{}) : dispatch(__half{});
  return e == cudaSuccess ? MSGL_OK : cuda_fail("paged_prefill_attention_q4", e);
}

}  // extern "C"
