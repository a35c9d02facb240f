// Paged attention for few query rows per sequence over the 4-bit pool (kv4.cuh): flash decoding over equal shares of a batch.
//
// Columns.  What shares a KV head of a sequence are its columns: the group of query heads of one token (decode), or of each of a
// few new tokens (BLOCKS: a verify or draft block, under the masks of the prefill op).  A CTA takes 8 NT of them; with more
// there are several CTAs for a share, side by side, and the second one's blocks come out of L2.
//
// Work split.  For every KV head the sequences' 16-token blocks are laid end to end and cut into equal shares; a CTA owns one
// share of one head.  The part of a sequence that a share holds is a segment; a segment that is a whole sequence writes final
// rows, any other an fp32 partial (weighted sum, maximum, sum of the weights), and the CTA that arrives last at the
// (sequence, head)'s counter merges its pieces.  One launch.
//
// A block of a head (codes, scales and biases of K: 9 head_dim bytes, and of V) is contiguous.  The warps of a CTA take the blocks of
// a segment in turn, U at a step, into a ring of their own; the pool is a tensor of rows of 1152 bytes, so a step's four rows of K come with
// one tile::gather4 load, and as many of V (rows past the tensor's end, for blocks that are not there and pages that are not in
// the pool, read as zeros, i.e. as zero keys and values).  A copy instruction costs its warp 67 to 93 cycles, and with one for
// every block of K and of V a fifth of the loop was that.
//
// Arithmetic.  The codes go to the tensor cores as they are, because small integers are f16 numbers already: the pattern n 2^k, inside
// the fraction, is n 2^(k-24).  A word masked, shifted by eight and masked, gives its elements two by two.
//   S = K q^T:    m16n8k16 with 16 tokens as rows and 8 columns.  k steps stay inside a group of 64 elements, so
//                 s = sum_g scale_g (sum_d n q) + bias_g sum_d q, in fp32.  q is an f16 number times a power of two of its row
//                 (exactly, but for what is below 2^-24 of the row's largest).
//   O^T = V^T P^T: rows are head_dim, the 16 tokens the k dimension.  A group's scale belongs to the token, so it is multiplied
//                 into the weight: P_g = f16(p scale_g f), and sum(p bias_g) is kept in fp32.  That rounding of P_g, half a unit
//                 of f16, is the only one in front of the output's.  f is a power of two of the column and the group that puts
//                 the largest p scale_g so far to 1/2 .. 2^15: groups of any size, and tokens of any size whose weight is small, leave
//                 each other their bits (eleven down to 2^-13 of the largest, below that 2^-24 of it).
// (Columns as rows and tokens as columns, the usual way round, leaves half of each product's rows empty at eight columns; to
// scale the codes to 16-bit values first takes twice the integer instructions, and rounds every element.  The byte n is the e4m3 number
// n 2^-9 and would take half the masks, but a product of e4m3 with an fp32 sum is made of two of f16, conversions and additions
// here: 171 us for 32 requests of 4096 to 32768 tokens.)
// The weights' reference maximum, a whole number, moves only when a score passes it by more than 2^8, and f when p scale_g could pass
// 2^15 / f by the largest of both in a lane, so that maxima need not be reduced in every step.
//
// What bounds it: no one pipe; integer instructions that take the codes apart (52 % of that pipe, as of the issue slots), by eight warps an SM, next
// to the memory.  32 requests of 4096 to 32768 tokens, 8 KV heads of 128, four query heads each: 111 to 116 us behind a write of the whole
// L2, 109 without, 4.4 to 4.7 TB/s (the same over 16-bit pages: 290; with one power of two for all scales 108 and 99).  At head_dim 256 a
// warp's sums leave two warps a quarter: 19 requests of 512 to 16384 tokens, two KV heads, 30 us, 20 of them start, ends and merges
// around a loop of six steps; at few tokens the launch (700 tokens 8.4 us, the 16-bit operator 8.3).
#pragma once

#include "kv4.cuh"

namespace msgl {

struct Q4DecodeParams {
  const void* q;              // (rows, hq, D)
  const unsigned char *k_pool, *v_pool;
  const int32_t *page_indptr, *page_indices, *kv_lens;
  const int32_t *qo_indptr, *prefix_lens;   // BLOCKS
  int total_q;                // BLOCKS: rows of q
  int page_blocks;            // blocks of 16 tokens per page
  int total_pages;            // entries of page_indices
  void* out;
  const void* gate;           // like q, or null
  // (2 shares, hkv, column tiles, 8 NT, D + 4) partials: weighted sums, maximum, sum of the weights.  Row 2 s of share s is the
  // end or a middle part of a sequence that began in front of it, row 2 s + 1 the first part of one that goes on behind it.
  float* part;
  int* tickets;               // (batch, hkv, column tiles) arrival counters, zero before and after
  int* status;
  int batch, hq, hkv, group;
  int col_tiles;              // CTAs side by side
  int num_shares;             // per head
  int min_share, pad;         // blocks a share holds at least; blocks that the end of a segment counts for
  int is_cross, window;       // BLOCKS
  int64_t num_blocks;
  int num_rows;               // of the pools as tensors
  float scale_log2;
};

__host__ __device__ constexpr int q4_merge_row(int hd) { return hd + 4; }
__host__ __device__ constexpr int q4_partial_floats(int hd) { return hd + 4; }
__host__ __device__ constexpr int q4_decode_smem(int hd, int warps, int stages) {
  return warps * stages * 2 * kv4_block_bytes(hd) + warps * 8 * q4_merge_row(hd) * 4 + warps * 16 * 4;
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// U blocks a step and stage: with two, the next block's loads and products fill the first one's waits.
template <typename T, int HD, int NT, bool BLOCKS, int U, int WARPS, int STAGES, int MINB>
__global__ void __launch_bounds__(WARPS * 32, MINB)
    q4_decode_kernel(const Q4DecodeParams p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  constexpr int G = HD / kKv4Group;          // groups of a row
  constexpr int BLK = kv4_block_bytes(HD);
  constexpr int ROW = HD / 2;                // code bytes of a row
  constexpr int PAIRS = kv4_pairs_at(HD);
  constexpr int MROW = q4_merge_row(HD), PROW = q4_partial_floats(HD);
  constexpr int COLS = 8 * NT;
  constexpr bool GATHER = U * HD == 512;     // four rows of the tensor a step (else: bulk copies)
  constexpr int WORDS = 2 * G;               // words of a K row per lane
  // f16 outputs: sum P_g n + p bias as sum P_g (n - 7.5) + (p bias + 7.5 P_g), with the rounded P_g in both, so that its rounding counts by
  // the distance from the middle code, 3 on the average for 8 (0.00035 to 0.00041 off 64 bits as a norm without it, where
  // the rounding of the output is 0.00021; bf16's is 0.0016).
  constexpr bool CENTRED = std::is_same<T, __half>::value;
  constexpr float kSlack = 8.f;
  constexpr float kNoScore = -1.5e38f;       // reference maximum of a column without a key (its sums are zero)
  constexpr float kMostFactor = 110.f;       // log2 of f at most
  constexpr float kNoFactor = 8.077935669463161e-28f;      // 2^-90: f of a column without a key
  using Mma = MmaOp<__half>;

  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ uint64_t s_bar[WARPS * STAGES];
  __shared__ int s_last[2];
  struct Keys {
    int page0, len;      // its first page, its tokens (clamped to what the pages hold)
    int first, blocks;   // blocks with a key that some of its columns see
    int tok0, new_tok;   // BLOCKS: first query token and how many
    int prefix;
  };
  struct Segment {
    Keys k;
    int beg;             // position of the whole sequence
    int lo, ng;          // first of its blocks in the share, and how many
    int cols;            // columns of this CTA
  };
  // (what a warp needs now and then does not sit in its registers)
  struct Ahead {
    Segment s;
    int b, step, more;
  };
  __shared__ Ahead s_ahead[WARPS];
  __shared__ Segment s_current[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, c = lane & 3;
  const int h = static_cast<int>(blockIdx.x) % p.hkv;
  const int ct = BLOCKS || COLS < 16 ? static_cast<int>(blockIdx.x) / p.hkv % p.col_tiles : 0;
  const int share_id = static_cast<int>(blockIdx.x) / p.hkv / p.col_tiles;
  unsigned char* const ring = smem_raw + warp * (STAGES * U * 2 * BLK);
  float* const sm_o = reinterpret_cast<float*>(smem_raw + WARPS * STAGES * U * 2 * BLK);   // [WARPS][8][MROW]
  float* const sm_ml = sm_o + WARPS * 8 * MROW;                                       // [WARPS][8][2]
  if (lane < STAGES) mbar_init(smem_u32(&s_bar[warp * STAGES + lane]), 1);
  if (GATHER && tid == 0 && p.num_rows > 0) {       // (no maps over a pool without slots)
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  fence_mbar_init();
  __syncwarp();
  grid_dependency_wait();
  grid_dependency_launch();
  const int32_t* const indptr = after_wait(p.page_indptr);
  const int32_t* const pages = after_wait(p.page_indices);
  const int32_t* const lens = after_wait(p.kv_lens);
  const int32_t* const new_tokens = BLOCKS ? after_wait(p.qo_indptr) : nullptr;
  const int32_t* const prefixes = BLOCKS ? after_wait(p.prefix_lens) : nullptr;
  const T* const q = after_wait(static_cast<const T*>(p.q));
  const unsigned char* const kp = after_wait(p.k_pool);
  const unsigned char* const vp = after_wait(p.v_pool);

  // ---- positions: a sequence takes its blocks and `pad` more; this CTA has [r0, r1)
  auto keys = [&](int b) -> Keys {
    Keys k{};
    k.page0 = min(max(__ldg(indptr + b), 0), p.total_pages);
    const int last = min(__ldg(indptr + b + 1), p.total_pages);
    const int64_t cap = static_cast<int64_t>(max(last - k.page0, 0)) * p.page_blocks * kKv4Rows;
    k.len = static_cast<int>(min(static_cast<int64_t>(max(__ldg(lens + b), 0)), cap));
    k.first = 0;
    if constexpr (BLOCKS) {
      k.tok0 = min(max(__ldg(new_tokens + b), 0), p.total_q);
      k.new_tok = max(min(__ldg(new_tokens + b + 1), p.total_q) - k.tok0, 0);
      k.prefix = __ldg(prefixes + b);
      const int hi = p.is_cross ? k.len : static_cast<int>(min(static_cast<int64_t>(k.len), static_cast<int64_t>(k.prefix) + k.new_tok));
      const int lo = p.window > 0 ? max(0, k.prefix - p.window + 1) : 0;
      k.first = lo / kKv4Rows;
      k.blocks = hi > lo && k.new_tok > 0 ? (hi + kKv4Rows - 1) / kKv4Rows - k.first : 0;
    } else {
      k.blocks = (k.len + kKv4Rows - 1) / kKv4Rows;
    }
    return k;
  };
  auto room = [&](int blocks) -> int { return blocks == 0 ? 0 : blocks + p.pad; };
  const int run = (p.batch + 31) / 32;
  int sum = 0;
  for (int j = 0; j < run; ++j) {
    const int b = lane * run + j;
    if (b < p.batch) sum = min(sum + room(keys(b).blocks), 1 << 28);
  }
  // (All pages of a call hold less than 2^27 blocks.  Row pointers that lay more end to end are none of a batch: no positions for
  // them, and zeros for the rows.)
  if (__reduce_add_sync(0xffffffffu, sum >> 8) > 1 << 20) {
    if (blockIdx.x == 0 && tid == 0 && p.status) atomicOr(p.status, 2);
    const int64_t pieces = static_cast<int64_t>(BLOCKS ? p.total_q : p.batch) * p.hq * (HD / 8);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * (WARPS * 32) + tid; i < pieces; i += static_cast<int64_t>(gridDim.x) * (WARPS * 32))
      static_cast<uint4*>(p.out)[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  const int total = __shfl_sync(0xffffffffu, incl, 31);
  const int share = max(p.min_share, (total + p.num_shares - 1) / p.num_shares);
  const int64_t start = static_cast<int64_t>(share_id) * share;
  if (start >= total && share_id > 0) return;
  const int r0 = static_cast<int>(start);
  const bool tail = start + share >= total;          // empty sequences at the end are this one's too
  const int r1 = tail ? total : r0 + share;
  // first sequence that starts at r0 or holds it
  int b0, beg0;
  {
    const int l = __ffs(__ballot_sync(0xffffffffu, incl >= r0)) - 1;
    int found = min(l * run + run, p.batch), at = incl;
    if (lane == l) {
      int pos = incl - sum;
      for (int j = 0; j < run; ++j) {
        const int b = l * run + j;
        if (b >= p.batch) break;
        const int n = room(keys(b).blocks);
        if (pos >= r0 || pos + n > r0) {
          found = b;
          at = pos;
          break;
        }
        pos += n;
      }
    }
    b0 = __shfl_sync(0xffffffffu, found, l);
    beg0 = __shfl_sync(0xffffffffu, at, l);
  }

  auto segment = [&](int b, int beg, Segment& s) -> bool {
    if (b >= p.batch || (beg >= r1 && !tail)) return false;
    s.beg = beg;
    s.k = keys(b);
    const int lo = max(beg, r0), hi = min(beg + s.k.blocks, r1);
    s.lo = lo - beg;
    s.cols = min((BLOCKS ? s.k.new_tok : 1) * p.group - ct * COLS, COLS);
    s.ng = s.cols > 0 ? max(hi - lo, 0) : 0;
    return true;
  };
  auto behind = [&](const Segment& s) -> int { return s.beg + room(s.k.blocks); };

  // ---- copies, ahead of the arithmetic: this warp's steps of the share in order.  The lanes hold the blocks of the next
  // 32 / U steps, U lanes a step: -1 a page that is not in the pool, -2 none.
  constexpr int BATCH = 32 / U;
  constexpr uint32_t ALL = (1u << U) - 1;
  Segment cs;
  bool go = segment(b0, beg0, cs);
  if (lane == 0) s_ahead[warp] = Ahead{cs, b0, warp, go};
  __syncwarp();
  // query row of a column of this CTA
  auto row_of = [&](int b, int tok0, int col) -> int64_t {
    if constexpr (!BLOCKS) return static_cast<int64_t>(b) * p.hq + h * p.group + ct * COLS + col;
    const int n = ct * COLS + col, t = n / p.group;
    return static_cast<int64_t>(tok0 + t) * p.hq + h * p.group + (n - t * p.group);
  };
  // a segment's q as it is, word (r8, g) = (2 c + w / G, w % G) of a lane's column; the first one's on its way under the page ids
  uint32_t qf[NT][WORDS][4];
  auto fetch_q = [&](int b) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = nt * 8 + r;
      const T* qr = q + (col < cs.cols ? row_of(b, cs.k.tok0, col) : 0) * HD + 16 * c;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (col < cs.cols) x = __ldg(reinterpret_cast<const uint4*>(qr + (w % G) * 64 + (w / G) * 8));
        qf[nt][w][0] = x.x;
        qf[nt][w][1] = x.y;
        qf[nt][w][2] = x.z;
        qf[nt][w][3] = x.w;
      }
    }
  };
  if (go) fetch_q(b0);
  int have = 0, at = 0;            // steps of this batch, next one
  int my_block = -2;
  uint32_t bad = 0;                // blocks in the ring whose page is not in the pool
  auto refill = [&]() {
    Ahead a = s_ahead[warp];
    while (true) {
      if (!a.more) break;
      const int steps = (a.s.ng + U - 1) / U;
      if (a.step < steps) {
        have = min(BATCH, (steps - a.step + WARPS - 1) / WARPS);
        break;
      }
      a.step -= steps;
      a.more = segment(++a.b, behind(a.s), a.s);
    }
    my_block = -2;
    if (a.more) {
      at = 0;
      const int i = (a.step + lane / U * WARPS) * U + lane % U;
      if (lane / U < have && i < a.s.ng) {
        const int g = a.s.k.first + a.s.lo + i;
        const int page = p.page_blocks == 1 ? g : g / p.page_blocks;
        const int64_t block = static_cast<int64_t>(__ldg(pages + a.s.k.page0 + page)) * p.page_blocks + (g - page * p.page_blocks);
        my_block = block >= 0 && block < p.num_blocks ? static_cast<int>(block) : -1;
        if (my_block < 0 && p.status) atomicOr(p.status, 2);
      }
      a.step += have * WARPS;
    }
    __syncwarp();
    if (lane == 0) s_ahead[warp] = a;
    __syncwarp();
    return a.more != 0;
  };
  const int64_t block_bytes = static_cast<int64_t>(p.hkv) * BLK, head_at = static_cast<int64_t>(h) * BLK;
  auto issue = [&](int stage) {    // this warp's next step into a stage, if it has one: its blocks of K, then of V
    if (at == have && !refill()) return;
    const uint32_t bar = smem_u32(&s_bar[warp * STAGES + stage]);
    const uint32_t dst = smem_u32(ring) + stage * (2 * U * BLK);
    if constexpr (GATHER) {
      constexpr int PARTS = 4 / U;           // rows of the tensor a block
      int row[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int block = __shfl_sync(0xffffffffu, my_block, at * U + i / PARTS);
        row[i] = block < 0 ? p.num_rows : (block * p.hkv + h) * PARTS + i % PARTS;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, 2 * U * BLK);
        tma_gather4(dst, &tm_k, row, bar);
        tma_gather4(dst + U * BLK, &tm_v, row, bar);
      }
    } else {
      const int block = __shfl_sync(0xffffffffu, my_block, at * U + lane % U);
      const uint32_t in = __ballot_sync(0xffffffffu, block >= 0) & ALL;
      if (bad != 0 || in != ALL) {
        const uint32_t out = __ballot_sync(0xffffffffu, block == -1) & ALL;
        bad = (bad & ~(ALL << (stage * U))) | out << (stage * U);
      }
      if (lane == 0) mbar_arrive_expect_tx(bar, __popc(in) * (2 * BLK));
      if (lane < U && block >= 0) {
        const int64_t off = block * block_bytes + head_at;
        bulk_load(dst + lane * BLK, kp + off, BLK, bar);
        bulk_load(dst + (U + lane) * BLK, vp + off, BLK, bar);
      }
    }
    ++at;
  };
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i) issue(i);
  int stage = 0;
  uint32_t parity = 0;

  bool alive = true;
  int part_b[2] = {0, 0}, part_first[2] = {0, 0}, part_count[2] = {0, 0}, parts = 0;
  const int rho = r ^ (r >> 1 & 1);          // token of row r: with 64-byte rows, the four tokens that lanes of a column read
                                             // of V then lie in two bank halves
  const int tv = 2 * c + (c & 1), tw = 2 * c + 1 - (c & 1);   // tokens of k index 2 c and 2 c + 1
  int cg = warp;
  for (int b = b0; go; go = segment(b + 1, behind(cs), cs), ++b) {
    if (h == 0 && ct == 0 && tid == 0 && cs.beg >= r0 && p.status && __ldg(lens + b) != cs.k.len)
      atomicOr(p.status, 2);    // a length that is negative or beyond the sequence's pages: clamped, reported
    if (BLOCKS && h == 0 && ct == 0 && tid == 0 && cs.beg >= r0 && p.status &&
        static_cast<int64_t>(cs.k.new_tok) * p.group > p.col_tiles * COLS)
      atomicOr(p.status, 2);    // more new tokens than the call was told of: the rows behind are not written
    if (cs.cols <= 0 || (cs.ng == 0 && cs.k.blocks > 0)) continue;
    if (lane == 0) s_current[warp] = cs;
    __syncwarp();
    if (b != b0) fetch_q(b);
    // ---- q: B fragments of the k steps (two of a word), 16 times q where the codes are the lowest bits of the fraction, and
    // a group's sum of q (2^-20 of it, as the products have it) for this lane's two columns
    float qs[NT][G][2], cscale[NT][2];
    int tok[NT][2];          // BLOCKS: token of this lane's columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < WORDS; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(qf[nt][w][i] >> 16 & 0x7fffu, qf[nt][w][i] & 0x7fffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float power = row_power(T{}, top), inv = power_inverse(power);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        cscale[nt][j] = p.scale_log2 * 1048576.f * __shfl_sync(0xffffffffu, power, (2 * c + j) * 4);
        tok[nt][j] = BLOCKS ? (ct * COLS + nt * 8 + 2 * c + j) / p.group : 0;
      }
#pragma unroll
      for (int w = 0; w < WORDS; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = unpack_pair(T{}, qf[nt][w][i]);
          const float by = i & 1 ? inv : 16.f * inv;
          qf[nt][w][i] = Mma::pack(x.x * by, x.y * by);
        }
      const uint32_t unit[4] = {0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u};
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float one[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = g; w < WORDS; w += G)
#pragma unroll
          for (int i = 0; i < 4; i += 2) Mma::run(one, unit, qf[nt][w][i], qf[nt][w][i + 1]);
        qs[nt][g][0] = one[0];
        qs[nt][g][1] = one[1];
      }
    }
    // tokens of the segment, and those that every column sees (BLOCKS: from the last token's window to the first token's position)
    const int t_lo = (cs.k.first + cs.lo) * kKv4Rows;
    const int t_hi = min(cs.k.len, (cs.k.first + cs.lo + cs.ng) * kKv4Rows);
    const int all_lo = BLOCKS && p.window > 0 ? cs.k.prefix + cs.k.new_tok - p.window : 0;
    const int all_hi = BLOCKS && !p.is_cross ? min(t_hi, cs.k.prefix + 1) : t_hi;
    const int steps = (cs.ng + U - 1) / U, prefix = cs.k.prefix;
    float o[NT][G][4][4];        // [group][nibble]: elements 64 g + 8 r + 2 i, + 1 of columns 2 c, 2 c + 1
    float pbias[NT][G][2];       // sums of p bias_g over this lane's tokens
    float m[NT][2], l[NT][2];
    float f[NT][G][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        f[nt][g][0] = f[nt][g][1] = kNoFactor;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][g][i][e] = 0.f;
        }
        pbias[nt][g][0] = pbias[nt][g][1] = 0.f;
      }
      m[nt][0] = m[nt][1] = kNoScore;
      l[nt][0] = l[nt][1] = 0.f;
    }

#pragma unroll 1
    for (; cg < steps; cg += WARPS) {
      const uint32_t bar = smem_u32(&s_bar[warp * STAGES + stage]);
      if (__any_sync(0xffffffffu, !mbar_try_wait(bar, parity))) {
        if (!alive) continue;
        bool ok;
        const long long t0 = clock64();
        while (!(ok = mbar_try_wait(bar, parity)) && clock64() - t0 < kTcWaitCycles) {
        }
        alive = __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
        if (!alive) continue;
      }
      const unsigned char* const step_at = ring + stage * (U * 2 * BLK);
      const int t0 = t_lo + cg * (U * kKv4Rows);
      auto step = [&](auto blocks) {
        constexpr int N = decltype(blocks)::value;
        // pairs of tokens rho and rho + 8
        uint32_t kpair[N][2][G], vpair[N][2][G];
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const unsigned char* at = step_at + u * BLK + PAIRS + (rho + 8 * t) * (G * 4);
            read_words<G * 4>(kpair[u][t], at);
            read_words<G * 4>(vpair[u][t], at + U * BLK);
          }
        if (t0 + N * kKv4Rows > t_hi || (!GATHER && bad != 0)) {   // rows behind the end hold anything; a page outside the pool: zeros
#pragma unroll
          for (int u = 0; u < N; ++u)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (t0 + u * kKv4Rows + rho + 8 * t >= t_hi || (!GATHER && (bad >> (stage * U + u) & 1u))) {
#pragma unroll
                for (int g = 0; g < G; ++g) kpair[u][t][g] = vpair[u][t][g] = 0u;
              }
        }
        // ---- scores
        float s[N][NT][4];
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const unsigned char* const kb = step_at + u * BLK;
          uint32_t w0[WORDS], w1[WORDS];       // words of tokens rho and rho + 8
          read_words<4 * WORDS>(w0, kb + rho * ROW + c * (4 * WORDS));
          read_words<4 * WORDS>(w1, kb + (rho + 8) * ROW + c * (4 * WORDS));
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
            for (int w = g; w < WORDS; w += G) {
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                const uint32_t x = w0[w] >> (4 * i), y = w1[w] >> (4 * i);
                const uint32_t a[4] = {x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) Mma::run(acc[nt], a, qf[nt][w][i], qf[nt][w][i + 1]);
              }
            }
            const float2 p0 = unpack_pair(T{}, kpair[u][0][g]), p1 = unpack_pair(T{}, kpair[u][1][g]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                s[u][nt][j] = fmaf(p0.x, acc[nt][j], g == 0 ? p0.y * qs[nt][g][j] : fmaf(p0.y, qs[nt][g][j], s[u][nt][j]));
                s[u][nt][2 + j] = fmaf(p1.x, acc[nt][2 + j], g == 0 ? p1.y * qs[nt][g][j] : fmaf(p1.y, qs[nt][g][j], s[u][nt][2 + j]));
              }
            }
          }
        }
        float most = 0.f;          // p scale f is below this times 2^8
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float smax = 0.f, fmax = 0.f;
#pragma unroll
          for (int u = 0; u < N; ++u) smax = max3(smax, unpack_pair(T{}, vpair[u][0][g]).x, unpack_pair(T{}, vpair[u][1][g]).x);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) fmax = max3(fmax, f[nt][g][0], f[nt][g][1]);
          most = fmaxf(most, smax * fmax);
        }
        // ---- exponents over the reference (one that is not there yet is far below every score)
        float x[N][NT][4], over = -INFINITY;
        auto seen = [&](int u, int nt, int j) -> bool {
          const int t = t0 + u * kKv4Rows + rho + 8 * (j >> 1);
          if constexpr (!BLOCKS) return t < t_hi;
          const int pos = prefix + tok[nt][j & 1];
          return t < t_hi && (p.is_cross || t <= pos) && (p.window == 0 || t > pos - p.window);
        };
        const bool edge = t0 + N * kKv4Rows > all_hi || t0 < all_lo;
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[u][nt][j] *= cscale[nt][j & 1];
          }
        if (edge) {
#pragma unroll
          for (int u = 0; u < N; ++u)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) s[u][nt][j] = seen(u, nt, j) ? s[u][nt][j] : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][nt][j] = s[u][nt][j] - m[nt][j & 1];
            over = max3(max3(over, x[u][nt][0], x[u][nt][1]), x[u][nt][2], x[u][nt][3]);
          }
        if (__any_sync(0xffffffffu, over > kSlack || most > 128.f)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float mx = -INFINITY;
#pragma unroll
              for (int u = 0; u < N; ++u) mx = max3(mx, s[u][nt][j], s[u][nt][2 + j]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              mx = fmaxf(ceilf(mx), m[nt][j]);
              const float up = m[nt][j] - mx, a = fast_exp2(up);
              m[nt][j] = mx;
              l[nt][j] *= a;
#pragma unroll
              for (int u = 0; u < N; ++u) {
                x[u][nt][j] = s[u][nt][j] - mx;
                x[u][nt][2 + j] = s[u][nt][2 + j] - mx;
              }
#pragma unroll
              for (int g = 0; g < G; ++g) {
                pbias[nt][g][j] *= a;
                // the largest p scale of the step, and log2 of what the sums are in units of, as the new reference counts it
                float top = 0.f;
#pragma unroll
                for (int u = 0; u < N; ++u)
                  top = max3(top, fast_exp2(x[u][nt][j]) * unpack_pair(T{}, vpair[u][0][g]).x,
                             fast_exp2(x[u][nt][2 + j]) * unpack_pair(T{}, vpair[u][1][g]).x);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float e = static_cast<float>(static_cast<int>(__float_as_uint(top) >> 23) - 126);     // top < 2^e
                const float unit = 127.f - static_cast<float>(__float_as_uint(f[nt][g][j]) >> 23) + up;
                const float to = fmaxf(e > unit + 7.f ? e : unit, -kMostFactor);
                const float b = fast_exp2(unit - to);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  o[nt][g][i][j] *= b;
                  o[nt][g][i][2 + j] *= b;
                }
                f[nt][g][j] = mx == kNoScore ? kNoFactor : __uint_as_float(static_cast<uint32_t>(127 - static_cast<int>(to)) << 23);
              }
            }
          }
        }
        uint32_t pf[N][NT][G][2];      // P_g as B fragments
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][nt][j] = fast_exp2(x[u][nt][j]);
            l[nt][0] += x[u][nt][0] + x[u][nt][2];
            l[nt][1] += x[u][nt][1] + x[u][nt][3];
#pragma unroll
            for (int g = 0; g < G; ++g) {
              float2 p0 = unpack_pair(T{}, vpair[u][0][g]), p1 = unpack_pair(T{}, vpair[u][1][g]);
              const uint32_t w0 = Mma::pack(x[u][nt][0] * f[nt][g][0] * p0.x, x[u][nt][1] * f[nt][g][1] * p0.x);
              const uint32_t w1 = Mma::pack(x[u][nt][2] * f[nt][g][0] * p1.x, x[u][nt][3] * f[nt][g][1] * p1.x);
              if constexpr (CENTRED) {
                p0.y = fmaf(7.5f, p0.x, p0.y);
                p1.y = fmaf(7.5f, p1.x, p1.y);
                const float2 r0 = unpack_pair(T{}, w0), r1 = unpack_pair(T{}, w1);
                const float c0 = -7.5f * power_inverse(f[nt][g][0]), c1 = -7.5f * power_inverse(f[nt][g][1]);
                pbias[nt][g][0] = fmaf(c0, r0.x, fmaf(c0, r1.x, pbias[nt][g][0]));
                pbias[nt][g][1] = fmaf(c1, r0.y, fmaf(c1, r1.y, pbias[nt][g][1]));
              }
              pbias[nt][g][0] = fmaf(x[u][nt][0], p0.y, fmaf(x[u][nt][2], p1.y, pbias[nt][g][0]));
              pbias[nt][g][1] = fmaf(x[u][nt][1], p0.y, fmaf(x[u][nt][3], p1.y, pbias[nt][g][1]));
              pf[u][nt][g][0] = transpose_8x8(w0);
              pf[u][nt][g][1] = transpose_8x8(w1);
            }
          }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const unsigned char* const vb = step_at + (U + u) * BLK + r * (4 * G);
          uint32_t v0[G], v1[G], v2[G], v3[G];      // word r of tokens tv, tw, tv + 8, tw + 8
          read_words<4 * G>(v0, vb + tv * ROW);
          read_words<4 * G>(v1, vb + tw * ROW);
          read_words<4 * G>(v2, vb + (tv + 8) * ROW);
          read_words<4 * G>(v3, vb + (tw + 8) * ROW);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const uint32_t lo0 = __byte_perm(v0[g], v1[g], 0x5410), hi0 = __byte_perm(v0[g], v1[g], 0x7632);
            const uint32_t lo1 = __byte_perm(v2[g], v3[g], 0x5410), hi1 = __byte_perm(v2[g], v3[g], 0x7632);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t mask = i & 1 ? 0x00f000f0u : 0x000f000fu;
              const uint32_t a[4] = {lo0 >> (8 * (i >> 1)) & mask, hi0 >> (8 * (i >> 1)) & mask, lo1 >> (8 * (i >> 1)) & mask,
                                     hi1 >> (8 * (i >> 1)) & mask};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) Mma::run(o[nt][g][i], a, pf[u][nt][g][0], pf[u][nt][g][1]);
            }
          }
        }
      };
      // (the last block of a segment, and the only one of a short sequence, by itself: a step of four takes 2900 cycles)
      if (U > 1 && t0 + kKv4Rows >= t_hi) step(std::integral_constant<int, 1>{});
      else step(std::integral_constant<int, U>{});
      __syncwarp();                 // every lane has read the stage: it is free
      issue(stage);
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
    }
    cg -= steps;
    cs = s_current[warp];

    // ---- end of the segment: the warps' sums are merged, eight columns at a time
    const bool whole = cs.ng == cs.k.blocks;
    const int64_t slot = (((2ll * share_id + (cs.beg >= r0 ? 1 : 0)) * p.hkv + h) * p.col_tiles + ct) * COLS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt * 8 >= cs.cols) break;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float lj = l[nt][j];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) lj += __shfl_xor_sync(0xffffffffu, lj, x);
        float* row = sm_o + (warp * 8 + 2 * c + j) * MROW + 8 * r;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float bj = pbias[nt][g][j];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) bj += __shfl_xor_sync(0xffffffffu, bj, x);
          float x[8];
          const float inv = power_inverse(f[nt][g][j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float unit = (i & 1 ? 1048576.f : 16777216.f) * inv;
            x[2 * i] = fmaf(o[nt][g][i][j], unit, bj);
            x[2 * i + 1] = fmaf(o[nt][g][i][2 + j], unit, bj);
          }
          *reinterpret_cast<float4*>(row + g * 64) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(row + g * 64 + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
        if (r == 0) *reinterpret_cast<float2*>(sm_ml + (warp * 8 + 2 * c + j) * 2) = make_float2(m[nt][j], lj);
      }
      __syncthreads();
#pragma unroll 1
      for (int e = tid; e < 2 * HD; e += WARPS * 32) {      // float4 pieces of the eight columns
        const int cc = e / (HD / 4), d = e % (HD / 4) * 4;
        const int col = nt * 8 + cc;
        if (col >= cs.cols) break;
        const int64_t at = row_of(b, cs.k.tok0, col) * HD + d;
        uint2 gate = make_uint2(0u, 0u);
        if (whole && p.gate != nullptr) gate = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.gate) + at);
        float M = -INFINITY, den = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm_ml[(w * 8 + cc) * 2]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float2 ml = *reinterpret_cast<const float2*>(sm_ml + (w * 8 + cc) * 2);
          const float wgt = fast_exp2(ml.x - M);
          den = fmaf(wgt, ml.y, den);
          const float4 y = *reinterpret_cast<const float4*>(sm_o + (w * 8 + cc) * MROW + d);
          x.x = fmaf(wgt, y.x, x.x);
          x.y = fmaf(wgt, y.y, x.y);
          x.z = fmaf(wgt, y.z, x.z);
          x.w = fmaf(wgt, y.w, x.w);
        }
        if (whole) {
          const float inv = den == 0.f ? 0.f : 1.f / den;
          uint2 y = make_uint2(MmaOp<T>::pack(x.x * inv, x.y * inv), MmaOp<T>::pack(x.z * inv, x.w * inv));
          if (p.gate != nullptr) y = make_uint2(apply_gate_pair<T>(y.x, gate.x), apply_gate_pair<T>(y.y, gate.y));
          *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at) = y;
        } else {
          float* to = p.part + (slot + col) * PROW;
          *reinterpret_cast<float4*>(to + d) = x;
          if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(M, den);
        }
      }
      __syncthreads();
    }
    if (!whole) {          // at most the first and the last segment of the share
      const int i = parts++ & 1;
      part_b[i] = b;
      part_first[i] = cs.beg / share;
      part_count[i] = (cs.beg + cs.k.blocks - 1) / share - part_first[i] + 1;
    }
  }

  // ---- the CTA that arrives last at a (sequence, head) merges its pieces
  if (tid < parts) {         // (a thread each: an arrival takes 2000 cycles)
    const int i = tid;
    int* ticket = p.tickets + (static_cast<int64_t>(part_b[i]) * p.hkv + h) * p.col_tiles + ct;
    s_last[i] = atomic_add_acq_rel(ticket, 1) == part_count[i] - 1;   // (the others' rows: behind the CTA barrier above)
    if (s_last[i]) *ticket = 0;
  }
  __syncthreads();
  for (int i = 0; i < parts; ++i) {
    if (s_last[i]) {
      const int64_t pitch = 2ll * p.hkv * p.col_tiles * COLS * PROW;          // from share to share
      const float* rows = p.part + part_first[i] * pitch + (static_cast<int64_t>(h) * p.col_tiles + ct) * COLS * PROW;
      const int n = part_count[i];
      const Keys k = keys(part_b[i]);
      const int cols = min((BLOCKS ? k.new_tok : 1) * p.group - ct * COLS, COLS);
      for (int e = tid; e < cols * (HD / 4); e += WARPS * 32) {
        const int col = e / (HD / 4), d = e % (HD / 4) * 4;
        const float* row = rows + col * PROW;
        const int head = BLOCKS ? (ct * COLS + col) % p.group : ct * COLS + col;
        const int64_t at = ((BLOCKS ? k.tok0 + (ct * COLS + col) / p.group : static_cast<int64_t>(part_b[i])) * p.hq + h * p.group + head) * HD + d;
        uint2 gate = make_uint2(0u, 0u);
        if (p.gate != nullptr) gate = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.gate) + at);
        auto piece = [&](int k) { return row + k * pitch + (k == 0 ? pitch / 2 : 0); };
        float M = -INFINITY, den = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int FLY = 8;                      // pieces in flight
#pragma unroll 1
        for (int k0 = 0; k0 < n; k0 += FLY) {
          float2 ml[FLY];
          float4 y[FLY];
#pragma unroll
          for (int k = 0; k < FLY; ++k) {
            const float* at = piece(min(k0 + k, n - 1));
            ml[k] = __ldcg(reinterpret_cast<const float2*>(at + HD));
            y[k] = __ldcg(reinterpret_cast<const float4*>(at + d));
          }
          float mx = M;
#pragma unroll
          for (int k = 0; k < FLY; ++k) mx = fmaxf(mx, ml[k].x);
          const float old = M == -INFINITY ? 0.f : fast_exp2(M - mx);
          M = mx;
          den *= old;
          x.x *= old;
          x.y *= old;
          x.z *= old;
          x.w *= old;
#pragma unroll
          for (int k = 0; k < FLY; ++k) {
            const float wgt = k0 + k >= n || ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - mx);
            den = fmaf(wgt, ml[k].y, den);
            x.x = fmaf(wgt, y[k].x, x.x);
            x.y = fmaf(wgt, y[k].y, x.y);
            x.z = fmaf(wgt, y[k].z, x.z);
            x.w = fmaf(wgt, y[k].w, x.w);
          }
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        uint2 y = make_uint2(MmaOp<T>::pack(x.x * inv, x.y * inv), MmaOp<T>::pack(x.z * inv, x.w * inv));
        if (p.gate != nullptr) y = make_uint2(apply_gate_pair<T>(y.x, gate.x), apply_gate_pair<T>(y.y, gate.y));
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at) = y;
      }
    }
  }
  if (!alive) {       // gave up: what is still on its way lands before the shared memory goes away; bounded
    if (p.status && lane == 0) atomicOr(p.status, 1);
    const long long t0 = clock64();
    for (int i = 0; i < STAGES; ++i) {
      while (!mbar_try_wait(smem_u32(&s_bar[warp * STAGES + stage]), parity) && clock64() - t0 < 2000000LL) {
      }
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
    }
  }
}

}  // namespace msgl
