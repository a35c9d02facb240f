// C-ABI entry points of the 4-bit K/V pool: rows in and out, norm + rotation + append, decode and prefill attention.
// Declarations: include/msgl_b200.h.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "decode_q4.cuh"
#include "host_common.cuh"
#include "kv4_project.cuh"
#include "prefill_pair.cuh"
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
  // (decode addresses a pool as rows of 1152 bytes, by 32 bits: 2.4 TB)
  if (num_slots / msgl::kKv4Rows * num_kv_heads * (head_dim / 128) >= (1ll << 31))
    return fail(MSGL_BAD_SHAPE, std::string(op) + "the pool has too many rows");
  return MSGL_OK;
}

// Groups of lanes that keep a B200 busy.
constexpr int64_t kItemsFill = 148 * 32;
// CTAs of 256 threads for so many threads' work, at most `per_sm` of them per SM (the kernels step through the rest).
unsigned grid_of(int64_t threads, int per_sm) {
  int sms = sm_count_cached();
  if (sms <= 0) sms = 148;
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, static_cast<int64_t>(sms) * per_sm)));
}

// ---- decode scheduling, in blocks of 16 tokens.  A share holds at least kQ4MinShare of them (4: geometric mean of twelve decode
// shapes, one to 61 sequences and 108 to 441093 tokens, 15.88 us, 8: 15.76, 16: 16.33), and the end of a segment counts for
// kQ4Pad (6: 17.0 us, 12: 15.76, 20: 15.68).  Batches of so many blocks that a wave's shares would be longer than kQ4MaxShare get
// whole waves more (2^31 tokens are then 131072 shares, and positions stay far from 32 bits).
constexpr int kQ4MinShare = 8;
constexpr int kQ4MaxShare = 1024;
constexpr int kQ4Pad = 20;

struct Q4Plan {
  int col_tiles, cols;       // CTAs side by side, columns of each
  int64_t shares;
  size_t ticket_bytes, part_bytes;
};
// `columns` of a sequence at most, `blocks` of all sequences at most.  Sixteen columns a CTA where a warp's registers hold
// them (head_dim 128): the second eight cost 375 cycles a block on top of 460, and 460 in a CTA of their own.
Q4Plan plan_q4(int batch, int columns, int hkv, int head_dim, int64_t blocks, int sms) {
  Q4Plan pl{};
  pl.cols = head_dim == 128 && columns > 8 ? 16 : 8;
  pl.col_tiles = (columns + pl.cols - 1) / pl.cols;
  const int ctas_per_sm = head_dim == 128 && pl.cols == 8 ? 2 : 1;
  const int64_t wave = std::max(1, sms * ctas_per_sm / (hkv * pl.col_tiles));
  blocks += static_cast<int64_t>(batch) * kQ4Pad;
  pl.shares = wave * std::max<int64_t>(1, (blocks + wave * kQ4MaxShare - 1) / (wave * kQ4MaxShare));
  const size_t tickets = static_cast<size_t>(batch) * hkv * pl.col_tiles;
  pl.ticket_bytes = tickets <= kTicketSlots ? 0 : (tickets * sizeof(int) + 255) / 256 * 256;
  pl.part_bytes = static_cast<size_t>(pl.shares) * 2 * hkv * pl.col_tiles * pl.cols * msgl::q4_partial_floats(head_dim) * sizeof(float);
  return pl;
}

template <typename T, int HD, int NT, bool BLOCKS, int U, int WARPS, int STAGES, int MINB>
cudaError_t launch_q4(const msgl::Q4DecodeParams& p, cudaStream_t s, const CUtensorMap& tm_k, const CUtensorMap& tm_v) {
  auto* kernel = msgl::q4_decode_kernel<T, HD, NT, BLOCKS, U, WARPS, STAGES, MINB>;
  constexpr int smem = msgl::q4_decode_smem(HD, WARPS, STAGES * U);
  const cudaError_t e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(p.num_shares * p.col_tiles * p.hkv)), dim3(WARPS * 32), smem, s, p, tm_k, tm_v);
}
// Blocks a step, warps, stages of the ring and CTAs per SM, by what fits (255 registers at eight warps an SM).  Eight columns of 128,
// 441093 tokens: 4 blocks, 4 warps, 2 CTAs 109 us; 2, 4, 3 CTAs 115; 4, 8, one CTA 125; 2, 12, one 129.  Head_dim 256, 97061
// tokens: 2 blocks, 8 warps, one CTA 29.3 us; 2, 4, two CTAs 32.1; 1, 12, one 33.9; 1, 4, three 38.4.  (Measured with
// a copy for each block, and one power of two for all scales; 109 and 27.4 us since.)  Sixteen columns: 2 blocks and a third stage, for their sums take twice the registers.
template <bool BLOCKS>
cudaError_t launch_q4_any(const msgl::Q4DecodeParams& p, int head_dim, int cols, int dtype, cudaStream_t s,
                          const CUtensorMap& tm_k, const CUtensorMap& tm_v) {
  auto go = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    if (head_dim == 256) return launch_q4<T, 256, 1, BLOCKS, 2, 8, 2, 1>(p, s, tm_k, tm_v);
    return cols == 8 ? launch_q4<T, 128, 1, BLOCKS, 4, 4, 2, 2>(p, s, tm_k, tm_v) : launch_q4<T, 128, 2, BLOCKS, 2, 8, 3, 1>(p, s, tm_k, tm_v);
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
  CUtensorMap tm_k, tm_v;
  std::memset(&tm_k, 0, sizeof(tm_k));
  std::memset(&tm_v, 0, sizeof(tm_v));
  const int64_t slots = p.num_blocks * msgl::kKv4Rows;
  if (slots == 0 && p.total_pages > 0) return fail(MSGL_BAD_SHAPE, std::string(op) + ": pages of a pool without slots");
  p.num_rows = static_cast<int>(p.num_blocks * p.hkv * (head_dim / 128));
  if (slots > 0 && (!make_pool_map(&tm_k, PoolBox::kPacked, p.k_pool, slots, p.hkv, head_dim, dtype) ||
                    !make_pool_map(&tm_v, PoolBox::kPacked, p.v_pool, slots, p.hkv, head_dim, dtype)))
    return fail(MSGL_CUDA_ERROR, std::string(op) + ": cannot build the tensor maps of the K/V pool");
  const cudaError_t e = launch_q4_any<BLOCKS>(p, head_dim, pl.cols, dtype, s, tm_k, tm_v);
  return e == cudaSuccess ? MSGL_OK : cuda_fail(op, e);
}

// Query blocks of few columns per KV head run the decode kernel (decode_q4.cuh), others the one-CTA tcgen05 kernel.  16 sequences of
// 16384 tokens, 8 KV heads, decode kernel / tcgen05: 8 columns 69 us / 222, 16 columns 115 / 222; with 20 to 64 columns as CTAs of
// 16 side by side, five verify tokens of 40 columns 81 / 63, draft blocks of 64 149 / 86 (60 and 78 since).
constexpr int kQ4BlockColumns = 16;
bool q4_block_form(int batch, int max_len_extend, int group) {
  return batch <= 65535 && static_cast<int64_t>(max_len_extend) * group <= kQ4BlockColumns;
}
// Blocks of a call at most: what the pages hold, or what a window leaves.
int64_t q4_block_bound(int batch, int64_t total_pages, int page_size, int max_len_extend, int window) {
  const int64_t all = total_pages * page_size / msgl::kKv4Rows;
  return window > 0 ? std::min<int64_t>(all, batch * ((static_cast<int64_t>(window) + max_len_extend) / msgl::kKv4Rows + 2)) : all;
}

// Long prefills lay their pages out first (kv4_expand_kernel) and run the pairs of CTAs, where those are the form for pages of 16
// bits and the attention takes several times what the copies do, by a rough model of both.  Sixty shapes (one to 24 sequences,
// 25 to 25650 new tokens, 176 to 180672 of keys, windows among them), time of the one-CTA form over time with expanded pages: at
// head_dim 128 where pairs are the form and the ratio is above 3, 1.03 to 1.21, below it 0.50 to 1.39, in the mean 0.93.  At head_dim
// 256 the one-CTA form has 128 rows and one CTA per SM, and 1.00 to 2.84 on all whose key range is not split and whose ratio is above
// 0.25.
constexpr size_t kQ4ExpandedMax = 256u << 20;     // bytes of pages
constexpr double kQ4ExpandWorth128 = 3.0, kQ4ExpandWorth256 = 0.25;
bool q4_expands(int batch, int total_q, int64_t total_kv, int hq, int hkv, int head_dim, int max_len_extend, bool cross,
                int window, int sms) {
  if (total_kv <= 0 || static_cast<size_t>(total_kv) * hkv * head_dim * 4 > kQ4ExpandedMax) return false;
  const PrefillPlan pl = plan_prefill(batch, total_q, total_kv, hq, hkv, head_dim, max_len_extend, window, sms);
  if (!prefill_pairs(batch, total_q, total_kv, hq / hkv, hkv, head_dim, max_len_extend, cross, window, pl.kv_chunk, true, sms))
    return false;
  double keys = std::max(1., static_cast<double>(total_kv) / batch - (cross ? 0. : 0.5 * total_q / batch));
  if (window > 0) keys = std::min<double>(keys, static_cast<double>(window) + max_len_extend);
  const double attend_us = 4. * head_dim * hq * static_cast<double>(total_q) * keys / 1e9;             // at 1 PFLOP/s
  const double copy_us = 5. + (static_cast<double>(total_kv) * hkv * 5.2 + static_cast<double>(total_q) * hq * 4.) * head_dim / 4e6;
  return attend_us > (head_dim == 256 ? kQ4ExpandWorth256 : kQ4ExpandWorth128) * copy_us;
}
// The largest numbers of every sequence and head (kv4_range_kernel), for long ones.
size_t q4_tops_bytes(int batch, int hkv) { return static_cast<size_t>(batch) * hkv * 2 * msgl::kRangeParts * sizeof(uint32_t); }
// CTAs of a sequence and head: about eight per SM in all.  (Thirty-two of each: 16 sequences of 8 heads under a window of 4096, 4 us more.)
int q4_range_parts(int batch, int hkv) {
  int parts = msgl::kRangeParts;
  while (parts > 1 && static_cast<int64_t>(batch) * hkv * parts > 148 * 8) parts /= 2;
  return parts;
}
msgl::Kv4ExpandParams q4_range_params(const void* k_cache, const void* v_cache, const int32_t* page_indices, const int32_t* page_indptr,
                                      const int32_t* kv_lens, const int32_t* prefix_lens, uint32_t* tops, int batch, int hkv,
                                      int64_t num_slots, int page_size, int64_t total_pages, int window) {
  msgl::Kv4ExpandParams x{};
  x.k_pool = static_cast<const unsigned char*>(k_cache);
  x.v_pool = static_cast<const unsigned char*>(v_cache);
  x.page_indices = page_indices;
  x.page_indptr = page_indptr;
  x.kv_lens = kv_lens;
  x.prefix_lens = prefix_lens;
  x.tops = tops;
  x.batch = batch;
  x.hkv = hkv;
  x.num_blocks = static_cast<int>(num_slots / msgl::kKv4Rows);
  x.page_blocks = page_size / msgl::kKv4Rows;
  x.total_pages = static_cast<int>(total_pages);
  x.window = window;
  x.parts = q4_range_parts(batch, hkv);
  return x;
}
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }
// K rows, V rows, sequences' powers, page ids, q rows and their powers.
size_t q4_expanded_bytes(int batch, int total_q, int64_t total_kv, int64_t total_pages, int hq, int hkv, int head_dim, int dtype) {
  const size_t rows = rounded(static_cast<size_t>(total_kv) * hkv * head_dim * 2);
  const size_t q_rows = static_cast<size_t>(total_q) * hq;
  return 2 * rows + q4_tops_bytes(batch, hkv) + rounded(total_pages * sizeof(int32_t)) +
         (dtype == MSGL_DTYPE_BF16 ? rounded(q_rows * head_dim * 2) + rounded(q_rows * sizeof(float)) : 0);
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
  if (static_cast<int64_t>(length) * num_kv_heads >= (1ll << 31))
    return fail(MSGL_BAD_SHAPE, std::string(op) + "too many rows for one call");
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
  p.hkv_recip = msgl::row_reciprocal(num_kv_heads);
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
  if (static_cast<int64_t>(length) * num_kv_heads >= (1ll << 31))
    return fail(MSGL_BAD_SHAPE, std::string(op) + "too many rows for one call");
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
  p.hkv_recip = msgl::row_reciprocal(num_kv_heads);
  p.status = static_cast<int*>(status_word);
  auto* kernel = head_dim == 256 ? (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_load_kernel<__nv_bfloat16, 256>
                                                             : msgl::kv4_load_kernel<__half, 256>)
                                 : (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_load_kernel<__nv_bfloat16, 128>
                                                             : msgl::kv4_load_kernel<__half, 128>);
  const cudaError_t e = launch_dependent(kernel, dim3(grid_of(static_cast<int64_t>(length) * num_kv_heads * head_dim / 16, 16)),
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
  // rows of an item: few while there are not items enough to fill the GPU, then as many as share a token's angles (8 q rows)
  const int64_t all_rows = static_cast<int64_t>(n_tokens) * (num_q_heads + 2 * num_kv_heads);
  int R = 1;
  while (R < 8 && all_rows > static_cast<int64_t>(R) * kItemsFill) R *= 2;
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
  p.item_rows = R;
  p.q_stride = q_token_stride;
  p.k_stride = k_token_stride;
  p.v_stride = v_token_stride;
  p.num_slots = num_slots;
  p.log2_base = std::log2(rope_base);
  p.eps = eps;
  p.minus_zero = -0.f;
  p.status = static_cast<int*>(status_word);
  auto* kernel = head_dim == 256 ? (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_project_kernel<__nv_bfloat16, 256>
                                                             : msgl::kv4_project_kernel<__half, 256>)
                                 : (dtype == MSGL_DTYPE_BF16 ? msgl::kv4_project_kernel<__nv_bfloat16, 128>
                                                             : msgl::kv4_project_kernel<__half, 128>);
  const cudaError_t e = launch_dependent(kernel, dim3(grid_of(items * msgl::kv4_project_lanes(head_dim), 4)), dim3(256), 0,
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
  if (!q4_block_form(batch, max_len_extend, group))
    return rounded(msgl_prefill_workspace_bytes(batch, total_q, total_pages * page_size, num_q_heads, num_kv_heads, head_dim,
                                                max_len_extend, sliding_window_size)) +
           q4_tops_bytes(batch, num_kv_heads);
  const int sms = sm_count_cached();
  const Q4Plan pl = plan_q4(batch, max_len_extend * group, num_kv_heads, head_dim,
                            q4_block_bound(batch, total_pages, page_size, max_len_extend, sliding_window_size), sms > 0 ? sms : 148);
  return kStatusBytes + pl.ticket_bytes + pl.part_bytes;
}

size_t msgl_prefill_expanded_bytes_q4(int batch, int total_q, int64_t total_pages, int page_size, int num_q_heads,
                                      int num_kv_heads, int head_dim, int dtype, int max_len_extend, int is_cross_attention,
                                      int sliding_window_size) {
  if (batch <= 0 || batch > 65535 || total_q <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      (head_dim != 128 && head_dim != 256) || total_pages < 0 || page_size <= 0 || total_pages >= (1ll << 31) / page_size)
    return 0;
  max_len_extend = std::max(1, max_len_extend);
  const int sms = sm_count_cached();
  const int64_t total_kv = total_pages * page_size;
  return q4_expands(batch, total_q, total_kv, num_q_heads, num_kv_heads, head_dim, max_len_extend, is_cross_attention != 0,
                    sliding_window_size, sms > 0 ? sms : 148)
             ? q4_expanded_bytes(batch, total_q, total_kv, total_pages, num_q_heads, num_kv_heads, head_dim, dtype)
             : 0;
}

int msgl_paged_prefill_attention_q4(const void* q, const void* k_cache, const void* v_cache, const int32_t* qo_indptr,
                                    const int32_t* page_indptr, const int32_t* page_indices, const int32_t* kv_lens,
                                    const int32_t* prefix_lens, const void* gate, void* out, void* workspace,
                                    size_t workspace_bytes, void* expanded, size_t expanded_bytes, int batch, int total_q, int num_q_heads, int num_kv_heads,
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
      !aligned16(workspace) || !aligned16(expanded))
    return fail(MSGL_BAD_ARG, std::string(op) + "q, the pools, out, gate and the workspace must be 16-byte aligned");
  const int sms = sm_count_cached();
  if (sms <= 0) return fail(MSGL_CUDA_ERROR, std::string(op) + "cannot query the device");
  if (q4_block_form(batch, max_len_extend, num_q_heads / num_kv_heads)) {
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
    p.total_q = total_q;
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
  const size_t used = rounded(kStatusBytes + pl.plan_bytes + pl.part_ml_bytes + pl.part_o_bytes);
  if (!workspace || workspace_bytes < used + q4_tops_bytes(batch, num_kv_heads))
    return fail(MSGL_BAD_ARG, std::string(op) + "workspace too small");
  if (static_cast<int64_t>(batch) * num_kv_heads > 0x7fffffffLL)
    return fail(MSGL_BAD_SHAPE, std::string(op) + "problem too large for one launch");
  const dim3 range_grid(static_cast<unsigned>(batch * num_kv_heads * q4_range_parts(batch, num_kv_heads)));
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
  const int64_t total_kv = total_pages * page_size;
  if (expanded != nullptr && batch <= 65535 &&
      q4_expands(batch, total_q, total_kv, num_q_heads, num_kv_heads, head_dim, max_len_extend, is_cross_attention != 0,
                 sliding_window_size, sms) &&
      expanded_bytes >= q4_expanded_bytes(batch, total_q, total_kv, total_pages, num_q_heads, num_kv_heads, head_dim, dtype)) {
    const int64_t pairs =
        msgl::prefill_item_bound(batch, total_q, total_kv, p.group, 256, max_len_extend, 0) * num_kv_heads;
    if (pairs * 2 > 0x7fffffffLL) return fail(MSGL_BAD_SHAPE, std::string(op) + "problem too large for one launch");
    const size_t rows = rounded(static_cast<size_t>(total_kv) * num_kv_heads * head_dim * 2);
    unsigned char* at = static_cast<unsigned char*>(expanded);
    msgl::Kv4ExpandParams x = q4_range_params(k_cache, v_cache, page_indices, page_indptr, kv_lens, prefix_lens,
                                              reinterpret_cast<uint32_t*>(at + 2 * rows), batch, num_kv_heads, num_slots, page_size,
                                              total_pages, sliding_window_size);
    x.k_rows = reinterpret_cast<__half*>(at);
    x.v_rows = reinterpret_cast<__half*>(at + rows);
    at += 2 * rows;
    at += q4_tops_bytes(batch, num_kv_heads);
    x.pages = reinterpret_cast<int32_t*>(at);
    at += rounded(total_pages * sizeof(int32_t));
    x.qo_indptr = qo_indptr;
    x.is_cross = is_cross_attention ? 1 : 0;
    x.status = p.status;
    const bool convert = dtype == MSGL_DTYPE_BF16;
    if (convert) {
      x.num_q_rows = static_cast<int64_t>(total_q) * num_q_heads;
      x.q = q;
      x.q_rows = reinterpret_cast<__half*>(at);
      x.q_power = reinterpret_cast<float*>(at + rounded(x.num_q_rows * head_dim * 2));
    }
    CUtensorMap tm_k, tm_v, tg_k, tg_v, tm_rows;
    const void* q16 = convert ? x.q_rows : q;
    if (!make_pool_map(&tm_k, PoolBox::kPage, x.k_rows, total_kv, num_kv_heads, head_dim, MSGL_DTYPE_F16) ||
        !make_pool_map(&tm_v, PoolBox::kPage, x.v_rows, total_kv, num_kv_heads, head_dim, MSGL_DTYPE_F16) ||
        !make_pool_map(&tg_k, PoolBox::kRow, x.k_rows, total_kv, num_kv_heads, head_dim, MSGL_DTYPE_F16) ||
        !make_pool_map(&tg_v, PoolBox::kRow, x.v_rows, total_kv, num_kv_heads, head_dim, MSGL_DTYPE_F16))
      return fail(MSGL_CUDA_ERROR, std::string(op) + "cannot build the tensor maps of the pages");
    p.q_tma = make_query_tensor_map(&tm_rows, q16, total_q, num_q_heads, p.group, head_dim, MSGL_DTYPE_F16) ? 1 : 0;
    if (!p.q_tma && !make_query_row_map(&tm_rows, q16, total_q, num_q_heads, head_dim, MSGL_DTYPE_F16))
      return fail(MSGL_CUDA_ERROR, std::string(op) + "cannot build the tensor map of the queries");
    p.q = q16;
    p.q_power = x.q_power;
    p.kv_tops = x.tops;
    p.k_cache = x.k_rows;
    p.v_cache = x.v_rows;
    p.page_indices = x.pages;
    p.num_slots = total_kv;
    p.kv_chunk = 0;
    p.chunk_recip = 0;
    auto run = [&](auto range, auto expand, auto kernel, int threads, int smem) -> cudaError_t {
      cudaError_t err = launch_dependent(range, range_grid, dim3(256), 0, s, x);
      if (err != cudaSuccess) return err;
      err = launch_dependent(expand, dim3(static_cast<unsigned>(sms * 8)), dim3(256), 0, s, x);
      if (err != cudaSuccess) return err;
      if ((err = allow_smem(kernel, smem)) != cudaSuccess) return err;
      return launch_clusters(2, kernel, dim3(static_cast<unsigned>(pairs * 2)), dim3(threads), smem, s, p, tm_k, tm_v, tg_k, tg_v,
                             tm_rows);
    };
    auto of = [&](auto tag) -> cudaError_t {
      using T = decltype(tag);
      using P128 = msgl::PairShape<128, true>;
      using P256 = msgl::PairShape<256, true>;
      return head_dim == 128 ? run(msgl::kv4_range_kernel<T, 128>, msgl::kv4_expand_kernel<T, 128>,
                                   msgl::prefill_pair_kernel<T, 128, true, __half, true>,
                                   P128::kThreads, P128::kSmemBytes)
                             : run(msgl::kv4_range_kernel<T, 256>, msgl::kv4_expand_kernel<T, 256>,
                                   msgl::prefill_pair_kernel<T, 256, true, __half, true>,
                                   P256::kThreads, P256::kSmemBytes);
    };
    const cudaError_t e = convert ? of(__nv_bfloat16{}) : of(__half{});
    return e == cudaSuccess ? MSGL_OK : cuda_fail("paged_prefill_attention_q4", e);
  }
  CUtensorMap none, tm_q;
  std::memset(&none, 0, sizeof(none));
  std::memset(&tm_q, 0, sizeof(tm_q));
  p.q_tma = make_query_tensor_map(&tm_q, q, total_q, num_q_heads, p.group, head_dim, dtype) ? 1 : 0;
  const dim3 grid(static_cast<unsigned>(pl.items * num_kv_heads));
  uint32_t* const tops = reinterpret_cast<uint32_t*>(ws + used);
  const bool range_first = head_dim == 128 && !prefill_short_q(max_len_extend, p.group, head_dim);      // (prefill_tc_kernel's OWN_RANGE)
  if (range_first) {
    p.kv_tops = tops;
    p.early = 1;          // what is older than the kernel in front is complete: the pool, q and the index arrays
  }
  auto launch = [&](auto range, auto kernel, auto merge, int threads, int smem) -> cudaError_t {
    cudaError_t err = allow_smem(kernel, smem);
    if (err != cudaSuccess) return err;
    if (range_first)
      err = launch_dependent(range, range_grid, dim3(256), 0, s,
                             q4_range_params(k_cache, v_cache, page_indices, page_indptr, kv_lens, prefix_lens, tops, batch, num_kv_heads,
                                             num_slots, page_size, total_pages, sliding_window_size));
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
      return launch(msgl::kv4_range_kernel<T, 256>, msgl::prefill_tc_kernel<T, 64, 1, 256, false, true>, msgl::prefill_merge_kernel<T, 256, S1w::kBM>,
                    S1w::kThreads, msgl::Kv4Shape<1, 256>::kSmemBytes);
    if (prefill_short_q(max_len_extend, p.group, head_dim))
      return launch(msgl::kv4_range_kernel<T, 128>, msgl::prefill_tc_kernel<T, 64, 1, 128, false, true>, msgl::prefill_merge_kernel<T, 128, S1::kBM>,
                    S1::kThreads, msgl::Kv4Shape<1, 128>::kSmemBytes);
    return launch(msgl::kv4_range_kernel<T, 128>, msgl::prefill_tc_kernel<T, 128, 2, 128, false, true>, msgl::prefill_merge_kernel<T, 128, S2::kBM>,
                  S2::kThreads, msgl::Kv4Shape<2, 128>::kSmemBytes);
  };
  const cudaError_t e = dtype == MSGL_DTYPE_BF16 ? dispatch(__nv_bfloat16{}) : dispatch(__half{});
  return e == cudaSuccess ? MSGL_OK : cuda_fail("paged_prefill_attention_q4", e);
}

}  // extern "C"
