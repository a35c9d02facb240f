// Paged attention for few query rows per sequence over the 4-bit pool (kv4.cuh): flash decoding over equal shares of a batch.
//
// Work split.  For every KV head the sequences' 16-token blocks are laid end to end and cut into equal shares; a CTA owns one
// share of one head.  The part of a sequence that a share holds is a segment; a segment that is a whole sequence writes final
// rows, any other an fp32 partial (weighted sum, maximum, sum of the weights), and the CTA that arrives last at the
// (sequence, head)'s counter merges its pieces.  One launch.
//
// A block of a head (codes, scales and biases of K: 9 head_dim bytes, and of V) comes with two bulk copies into a ring of the
// warp's own; the warps of a CTA take the blocks of a segment in turn.
//
// Arithmetic.  The codes go to the tensor cores as they are: a nibble put under the right exponent is the 16-bit
// number OFF + n, exactly, in one and-or, and what OFF adds is taken off in fp32:
//   S = K q^T:    m16n8k16 with 16 tokens as rows and 8 query heads as columns.  k steps stay inside a group of 64 elements, so
//                 s = sum_g scale_g (sum_d (OFF + n) q - sum_d OFF q) + bias_g sum_d q, with the middle term (per head and group,
//                 from a product with OFF itself) as the accumulator's start.
//   O^T = V^T P^T: rows are head_dim, the 16 tokens the k dimension.  A group's scale belongs to the token, so it is multiplied
//                 into the weight: P_g = T(p scale_g).  OFF sum(P_g) is taken off at the end (the sum by a product with ones),
//                 and sum(p bias_g) is kept in fp32.  T(p scale) is the one rounding in front of the output's: a relative half
//                 unit of T per weight, as a 16-bit pool's kernel rounds p.  It counts by the code, so codes are taken from their
//                 middle: with v = scale (n - 8) + (bias + 8 scale) its effect is 2.5 times less than with v = scale n + bias.
// (Heads as rows and tokens as columns, the usual way round, leaves half of each product's rows empty at eight heads; to
// scale the codes to 16-bit values first takes twice the integer instructions and rounds every element.)
// The weights' reference maximum moves only when a score passes it by more than 2^kSlack, so that the rows' maxima need not
// be reduced in every step.
#pragma once

#include "kv4.cuh"

namespace msgl {

struct Q4DecodeParams {
  const void* q;              // (rows, hq, D)
  const unsigned char *k_pool, *v_pool;
  const int32_t *page_indptr, *page_indices, *kv_lens;
  int page_blocks;            // blocks of 16 tokens per page
  int total_pages;            // entries of page_indices
  void* out;
  const void* gate;           // like q, or null
  // (2 shares, hkv, group, D + 4) partials: weighted sums, maximum, sum of the weights.  Row 2 s of share s is the end or a
  // middle part of a sequence that began in front of it, row 2 s + 1 the first part of one that goes on behind it.
  float* part;
  int* tickets;               // (batch, hkv) arrival counters, zero before and after
  int* status;
  int batch, hq, hkv, group;
  int num_shares;             // per head
  int min_share, pad;         // blocks a share holds at least; blocks that the end of a segment counts for
  int64_t num_blocks;
  float scale_log2;
};

__host__ __device__ constexpr int q4_merge_row(int hd) { return hd + 4; }
__host__ __device__ constexpr int q4_partial_floats(int hd) { return hd + 4; }
__host__ __device__ constexpr int q4_decode_smem(int hd, int warps, int stages) {
  return warps * stages * 2 * kv4_block_bytes(hd) + warps * 4 * q4_merge_row(hd) * 4 + warps * 8 * 4;
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
template <typename T, int HD, int NT, int WARPS, int STAGES, int MINB>
__global__ void __launch_bounds__(WARPS * 32, MINB) q4_decode_kernel(const Q4DecodeParams p) {
  constexpr int G = HD / kKv4Group;          // groups of a row
  constexpr int BLK = kv4_block_bytes(HD);
  constexpr int ROW = HD / 2;                // code bytes of a row
  constexpr int PAIRS = kv4_pairs_at(HD);
  constexpr int MROW = q4_merge_row(HD), PROW = q4_partial_floats(HD);
  using N = Nibble<T>;

  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ uint64_t s_bar[WARPS * STAGES];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, c = lane & 3;
  const int h = static_cast<int>(blockIdx.x) % p.hkv;
  const int share_id = static_cast<int>(blockIdx.x) / p.hkv;
  unsigned char* const ring = smem_raw + warp * (STAGES * 2 * BLK);
  float* const sm_o = reinterpret_cast<float*>(smem_raw + WARPS * STAGES * 2 * BLK);   // [WARPS][4][MROW]
  float* const sm_ml = sm_o + WARPS * 4 * MROW;                                       // [WARPS][4][2]
  if (lane < STAGES) mbar_init(smem_u32(&s_bar[warp * STAGES + lane]), 1);
  fence_mbar_init();
  __syncwarp();
  grid_dependency_wait();
  grid_dependency_launch();
  const int32_t* const indptr = after_wait(p.page_indptr);
  const int32_t* const pages = after_wait(p.page_indices);
  const int32_t* const lens = after_wait(p.kv_lens);
  const T* const q = after_wait(static_cast<const T*>(p.q));
  const unsigned char* const kp = after_wait(p.k_pool);
  const unsigned char* const vp = after_wait(p.v_pool);

  // ---- positions: a sequence takes its blocks and `pad` more; this CTA has [r0, r1)
  auto length = [&](int b, int& page0) -> int {      // tokens, clamped to what the sequence's pages hold
    page0 = min(max(__ldg(indptr + b), 0), p.total_pages);
    const int last = min(__ldg(indptr + b + 1), p.total_pages);
    const int64_t cap = static_cast<int64_t>(max(last - page0, 0)) * p.page_blocks * kKv4Rows;
    return static_cast<int>(min(static_cast<int64_t>(max(__ldg(lens + b), 0)), cap));
  };
  auto room = [&](int len) -> int { return len == 0 ? 0 : (len + kKv4Rows - 1) / kKv4Rows + p.pad; };
  const int run = (p.batch + 31) / 32;
  int sum = 0;
  for (int j = 0; j < run; ++j) {
    const int b = lane * run + j;
    int page0;
    if (b < p.batch) sum += room(length(b, page0));
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
        int page0;
        if (b >= p.batch) break;
        const int n = room(length(b, page0));
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

  struct Segment {
    int beg, ng_all;     // position and blocks of the whole sequence
    int lo, ng;          // first of its blocks in the share, and how many
    int page0, len;
  };
  auto segment = [&](int b, int beg, Segment& s) -> bool {
    if (b >= p.batch || (beg >= r1 && !tail)) return false;
    s.beg = beg;
    s.len = length(b, s.page0);
    s.ng_all = (s.len + kKv4Rows - 1) / kKv4Rows;
    const int lo = max(beg, r0), hi = min(beg + s.ng_all, r1);
    s.lo = lo - beg;
    s.ng = max(hi - lo, 0);
    return true;
  };
  auto behind = [&](const Segment& s) -> int { return s.beg + (s.ng_all == 0 ? 0 : s.ng_all + p.pad); };

  // ---- copies, ahead of the arithmetic: this warp's blocks of the share in order, 32 page ids at a time in the lanes
  Segment ps;
  int pb = b0, pg = warp;
  bool more = segment(pb, beg0, ps);
  int have = 0, at = 0;            // ids of this batch, next one
  int my_block = -1;
  uint32_t bad = 0;                // stages whose page is not in the pool
  auto issue = [&](int stage) {
    while (at == have) {
      if (!more) return;
      if (pg >= ps.ng) {
        pg -= ps.ng;
        more = segment(++pb, behind(ps), ps);
        continue;
      }
      have = min(32, (ps.ng - pg + WARPS - 1) / WARPS);
      at = 0;
      my_block = -1;
      if (lane < have) {
        const int g = ps.lo + pg + lane * WARPS;
        const int page = p.page_blocks == 1 ? g : g / p.page_blocks;
        const int64_t block = static_cast<int64_t>(__ldg(pages + ps.page0 + page)) * p.page_blocks + (g - page * p.page_blocks);
        if (block >= 0 && block < p.num_blocks) my_block = static_cast<int>(block);
        else if (p.status) atomicOr(p.status, 2);
      }
      pg += have * WARPS;
    }
    const int block = __shfl_sync(0xffffffffu, my_block, at++);
    bad = block < 0 ? bad | 1u << stage : bad & ~(1u << stage);
    if (lane == 0) {
      const uint32_t bar = smem_u32(&s_bar[warp * STAGES + stage]);
      if (block >= 0) {
        const int64_t off = (static_cast<int64_t>(block) * p.hkv + h) * BLK;
        const uint32_t dst = smem_u32(ring + stage * (2 * BLK));
        mbar_arrive_expect_tx(bar, 2 * BLK);
        bulk_load(dst, kp + off, BLK, bar);
        bulk_load(dst + BLK, vp + off, BLK, bar);
      } else {
        mbar_arrive(bar);
      }
    }
  };
  int stage = 0, fill = 0, ahead = 0;
  uint32_t parity = 0;
  auto top_up = [&]() {
#pragma unroll 1
    for (; ahead < STAGES; ++ahead) {
      issue(fill);
      fill = fill + 1 == STAGES ? 0 : fill + 1;
    }
  };
  top_up();

  bool alive = true;
  int part_b[2] = {0, 0}, part_first[2] = {0, 0}, part_count[2] = {0, 0}, parts = 0;
  const int rho = r ^ (r >> 1 & 1);          // token of row r: with 64-byte rows, the four tokens that lanes of a column read
                                             // of V then lie in two bank halves
  const int tv = 2 * c + (c & 1), tw = 2 * c + 1 - (c & 1);   // tokens of k index 2 c and 2 c + 1
  int cg = warp;
  Segment cs;
  for (int b = b0, beg = beg0; segment(b, beg, cs); beg = behind(cs), ++b) {
    if (h == 0 && tid == 0 && cs.beg >= r0 && p.status && __ldg(lens + b) != cs.len)
      atomicOr(p.status, 2);    // a length that is negative or beyond the sequence's pages: clamped, reported
    if (cs.ng == 0 && cs.ng_all > 0) continue;
    // ---- q: B fragments of a group's four k steps, and the group's sums of q and of OFF q for this lane's two columns
    uint32_t qf[NT][G][8];
    float qo[NT][G][2], qs[NT][G][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = nt * 8 + r;
      const T* qr = q + (static_cast<int64_t>(b) * p.hq + h * p.group + col) * HD + 16 * c;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
        if (col < p.group) {
          x = *reinterpret_cast<const uint4*>(qr + g * 64);
          y = *reinterpret_cast<const uint4*>(qr + g * 64 + 8);
        }
        qf[nt][g][0] = x.x;
        qf[nt][g][1] = x.y;
        qf[nt][g][2] = x.z;
        qf[nt][g][3] = x.w;
        qf[nt][g][4] = y.x;
        qf[nt][g][5] = y.y;
        qf[nt][g][6] = y.z;
        qf[nt][g][7] = y.w;
        float one[4] = {0.f, 0.f, 0.f, 0.f}, off[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t a1[4] = {both<T>(1.f), both<T>(1.f), both<T>(1.f), both<T>(1.f)};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const int i = 2 * (ks & 1);
          const uint32_t ao[4] = {both<T>(N::off(i)), both<T>(N::off(i)), both<T>(N::off(i + 1)), both<T>(N::off(i + 1))};
          MmaOp<T>::run(one, a1, qf[nt][g][2 * ks], qf[nt][g][2 * ks + 1]);
          MmaOp<T>::run(off, ao, qf[nt][g][2 * ks], qf[nt][g][2 * ks + 1]);
        }
        qs[nt][g][0] = one[0];
        qs[nt][g][1] = one[1];
        qo[nt][g][0] = -off[0];
        qo[nt][g][1] = -off[1];
      }
    }
    float o[NT][G][4][4];        // [group][nibble]: elements 64 g + 8 r + 2 i, + 1 of columns 2 c, 2 c + 1
    float ps4[NT][G][4];         // sums of P_g (elements 0 and 1)
    float pbias[NT][G][2];       // sums of p (bias_g + 8 scale_g) over this lane's tokens
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ps4[nt][g][e] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][g][i][e] = 0.f;
        }
        pbias[nt][g][0] = pbias[nt][g][1] = 0.f;
      }
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    for (; cg < cs.ng; cg += WARPS) {
      {
        const uint32_t bar = smem_u32(&s_bar[warp * STAGES + stage]);
        bool ok = !alive || mbar_try_wait(bar, parity);
        if (!ok) {
          const long long t0 = clock64();
          while (!(ok = mbar_try_wait(bar, parity)) && clock64() - t0 < kTcWaitCycles) {
          }
        }
        alive = __all_sync(0xffffffffu, alive && ok ? 1 : 0) != 0;
        if (!alive) continue;
      }
      const unsigned char* kb = ring + stage * (2 * BLK);
      const unsigned char* vb = kb + BLK;
      const int nvalid = cs.len - (cs.lo + cg) * kKv4Rows;       // >= 1
      // pairs of tokens rho and rho + 8
      uint32_t kpair[2][G], vpair[2][G];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        read_words<G * 4>(kpair[t], kb + PAIRS + (rho + 8 * t) * (G * 4));
        read_words<G * 4>(vpair[t], vb + PAIRS + (rho + 8 * t) * (G * 4));
      }
      if (nvalid < kKv4Rows || (bad >> stage & 1u)) {       // rows behind the end hold anything; a page outside the pool: zeros
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (rho + 8 * t >= nvalid || (bad >> stage & 1u)) {
#pragma unroll
            for (int g = 0; g < G; ++g) kpair[t][g] = vpair[t][g] = 0u;
          }
      }
      // ---- scores
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
      {
        uint32_t w0[2 * G], w1[2 * G];       // words 2 c (groups 0 .. G - 1) and 2 c + 1 of tokens rho and rho + 8
        read_words<8 * G>(w0, kb + rho * ROW + c * (8 * G));
        read_words<8 * G>(w1, kb + (rho + 8) * ROW + c * (8 * G));
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[nt][0] = acc[nt][2] = qo[nt][g][0];
            acc[nt][1] = acc[nt][3] = qo[nt][g][1];
          }
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint32_t x = w0[(ks >> 1) * G + g], y = w1[(ks >> 1) * G + g];
            const int i = 2 * (ks & 1);
            const uint32_t a[4] = {N::make(x, i), N::make(y, i), N::make(x, i + 1), N::make(y, i + 1)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) MmaOp<T>::run(acc[nt], a, qf[nt][g][2 * ks], qf[nt][g][2 * ks + 1]);
          }
          const float2 p0 = unpack_pair(T{}, kpair[0][g]), p1 = unpack_pair(T{}, kpair[1][g]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              s[nt][j] = fmaf(p0.y, qs[nt][g][j], fmaf(p0.x, acc[nt][j], s[nt][j]));
              s[nt][2 + j] = fmaf(p1.y, qs[nt][g][j], fmaf(p1.x, acc[nt][2 + j], s[nt][2 + j]));
            }
          }
        }
      }
      bool up = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[nt][j] *= p.scale_log2;
          if (nvalid < kKv4Rows && rho + 8 * (j >> 1) >= nvalid) s[nt][j] = -INFINITY;
          up |= s[nt][j] > m[nt][j & 1] + N::kSlack;
        }
      }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = fmaxf(s[nt][j], s[nt][2 + j]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            mx = fmaxf(mx, m[nt][j]);
            const float a = mx == -INFINITY ? 1.f : fast_exp2(m[nt][j] - mx);
            m[nt][j] = mx;
            l[nt][j] *= a;
#pragma unroll
            for (int g = 0; g < G; ++g) {
              pbias[nt][g][j] *= a;
              ps4[nt][g][j] *= a;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[nt][g][i][j] *= a;
                o[nt][g][i][2 + j] *= a;
              }
            }
          }
        }
      }
      uint32_t pf[NT][G][2];      // P_g as B fragments
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float mm = m[nt][j & 1];
          s[nt][j] = fast_exp2(s[nt][j] - (mm == -INFINITY ? 0.f : mm));
        }
        l[nt][0] += s[nt][0] + s[nt][2];
        l[nt][1] += s[nt][1] + s[nt][3];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float2 p0 = unpack_pair(T{}, vpair[0][g]), p1 = unpack_pair(T{}, vpair[1][g]);
          const float b0 = fmaf(8.f, p0.x, p0.y), b1 = fmaf(8.f, p1.x, p1.y);
          pbias[nt][g][0] = fmaf(s[nt][0], b0, fmaf(s[nt][2], b1, pbias[nt][g][0]));
          pbias[nt][g][1] = fmaf(s[nt][1], b0, fmaf(s[nt][3], b1, pbias[nt][g][1]));
          pf[nt][g][0] = transpose_8x8(MmaOp<T>::pack(s[nt][0] * p0.x, s[nt][1] * p0.x));
          pf[nt][g][1] = transpose_8x8(MmaOp<T>::pack(s[nt][2] * p1.x, s[nt][3] * p1.x));
        }
      }
      // ---- O^T += V^T P^T
      {
        uint32_t v0[G], v1[G], v2[G], v3[G];      // word r of tokens tv, tw, tv + 8, tw + 8
        read_words<4 * G>(v0, vb + tv * ROW + r * (4 * G));
        read_words<4 * G>(v1, vb + tw * ROW + r * (4 * G));
        read_words<4 * G>(v2, vb + (tv + 8) * ROW + r * (4 * G));
        read_words<4 * G>(v3, vb + (tw + 8) * ROW + r * (4 * G));
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t lo0 = __byte_perm(v0[g], v1[g], 0x5410), hi0 = __byte_perm(v0[g], v1[g], 0x7632);
          const uint32_t lo1 = __byte_perm(v2[g], v3[g], 0x5410), hi1 = __byte_perm(v2[g], v3[g], 0x7632);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {N::make(lo0, i), N::make(hi0, i), N::make(lo1, i), N::make(hi1, i)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) MmaOp<T>::run(o[nt][g][i], a, pf[nt][g][0], pf[nt][g][1]);
          }
          const uint32_t a1[4] = {both<T>(1.f), both<T>(1.f), both<T>(1.f), both<T>(1.f)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) MmaOp<T>::run(ps4[nt][g], a1, pf[nt][g][0], pf[nt][g][1]);
        }
      }
      __syncwarp();                 // every lane has read the stage
      --ahead;
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
      top_up();
    }
    cg -= cs.ng;

    // ---- end of the segment: the warps' sums are merged, four columns (those of one j) at a time
    const bool whole = cs.ng == cs.ng_all;
    const int64_t slot = ((2ll * share_id + (cs.beg >= r0 ? 1 : 0)) * p.hkv + h) * p.group;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (nt * 8 + j >= p.group) continue;         // (none of the columns 8 nt + j, + 2, + 4, + 6)
        float lj = l[nt][j];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) lj += __shfl_xor_sync(0xffffffffu, lj, x);
        float* row = sm_o + (warp * 4 + c) * MROW + 8 * r;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float bj = pbias[nt][g][j];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) bj += __shfl_xor_sync(0xffffffffu, bj, x);
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float d = fmaf(-8.f - N::off(i), ps4[nt][g][j], bj);
            x[2 * i] = o[nt][g][i][j] + d;
            x[2 * i + 1] = o[nt][g][i][2 + j] + d;
          }
          *reinterpret_cast<float4*>(row + g * 64) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(row + g * 64 + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
        if (r == 0) *reinterpret_cast<float2*>(sm_ml + (warp * 4 + c) * 2) = make_float2(m[nt][j], lj);
        __syncthreads();
        for (int e = tid; e < HD; e += WARPS * 32) {      // float4 pieces of the four columns
          const int cc = e / (HD / 4), d = e % (HD / 4) * 4;
          const int col = nt * 8 + 2 * cc + j;
          if (col >= p.group) continue;
          float M = -INFINITY, den = 0.f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm_ml[(w * 4 + cc) * 2]);
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WARPS; ++w) {
            const float mw = sm_ml[(w * 4 + cc) * 2];
            const float wgt = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
            den = fmaf(wgt, sm_ml[(w * 4 + cc) * 2 + 1], den);
            const float4 y = *reinterpret_cast<const float4*>(sm_o + (w * 4 + cc) * MROW + d);
            x.x = fmaf(wgt, y.x, x.x);
            x.y = fmaf(wgt, y.y, x.y);
            x.z = fmaf(wgt, y.z, x.z);
            x.w = fmaf(wgt, y.w, x.w);
          }
          if (whole) {
            const float inv = den == 0.f ? 0.f : 1.f / den;
            const int64_t at = (static_cast<int64_t>(b) * p.hq + h * p.group + col) * HD + d;
            alignas(8) T y[4] = {MmaOp<T>::from_float(x.x * inv), MmaOp<T>::from_float(x.y * inv),
                                 MmaOp<T>::from_float(x.z * inv), MmaOp<T>::from_float(x.w * inv)};
            if (p.gate != nullptr) {
#pragma unroll
              for (int k = 0; k < 4; ++k) y[k] = apply_gate<T>(to_f32(y[k]), static_cast<const T*>(p.gate)[at + k]);
            }
            *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at) = *reinterpret_cast<const uint2*>(y);
          } else {
            float* to = p.part + (slot + col) * PROW;
            *reinterpret_cast<float4*>(to + d) = x;
            if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(M, den);
          }
        }
        __syncthreads();
      }
    }
    if (!whole) {          // at most the first and the last segment of the share
      const int i = parts++ & 1;
      part_b[i] = b;
      part_first[i] = cs.beg / share;
      part_count[i] = (cs.beg + cs.ng_all - 1) / share - part_first[i] + 1;
    }
  }

  // ---- the CTA that arrives last at a (sequence, head) merges its pieces
  for (int i = 0; i < parts; ++i) {
    if (tid == 0) {
      int* ticket = p.tickets + static_cast<int64_t>(part_b[i]) * p.hkv + h;
      s_last = atomic_add_acq_rel(ticket, 1) == part_count[i] - 1;   // (the others' rows: behind the CTA barrier above)
      if (s_last) *ticket = 0;
    }
    __syncthreads();
    if (s_last) {
      const int64_t pitch = 2ll * p.hkv * p.group * PROW;          // from share to share
      const float* rows = p.part + part_first[i] * pitch + static_cast<int64_t>(h) * p.group * PROW;
      const int n = part_count[i];
      for (int e = tid; e < p.group * (HD / 4); e += WARPS * 32) {
        const int col = e / (HD / 4), d = e % (HD / 4) * 4;
        const float* row = rows + col * PROW;
        auto piece = [&](int k) { return row + k * pitch + (k == 0 ? pitch / 2 : 0); };
        float M = -INFINITY, den = 0.f;
#pragma unroll 4
        for (int k = 0; k < n; ++k) M = fmaxf(M, __ldcg(piece(k) + HD));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
          const float2 ml = __ldcg(reinterpret_cast<const float2*>(piece(k) + HD));
          const float4 y = __ldcg(reinterpret_cast<const float4*>(piece(k) + d));
          const float wgt = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
          den = fmaf(wgt, ml.y, den);
          x.x = fmaf(wgt, y.x, x.x);
          x.y = fmaf(wgt, y.y, x.y);
          x.z = fmaf(wgt, y.z, x.z);
          x.w = fmaf(wgt, y.w, x.w);
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const int64_t at = (static_cast<int64_t>(part_b[i]) * p.hq + h * p.group + col) * HD + d;
        alignas(8) T y[4] = {MmaOp<T>::from_float(x.x * inv), MmaOp<T>::from_float(x.y * inv),
                             MmaOp<T>::from_float(x.z * inv), MmaOp<T>::from_float(x.w * inv)};
        if (p.gate != nullptr) {
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = apply_gate<T>(to_f32(y[k]), static_cast<const T*>(p.gate)[at + k]);
        }
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at) = *reinterpret_cast<const uint2*>(y);
      }
    }
    __syncthreads();
  }
  if (!alive) {       // gave up: what is still on its way lands before the shared memory goes away; bounded
    if (p.status && lane == 0) atomicOr(p.status, 1);
    const long long t0 = clock64();
    for (; ahead > 0; --ahead) {
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
