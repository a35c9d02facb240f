// The K/V pool held in 4 bits: its format, and the kernels that put rows into it and read them back.
//
// Sixteen slots are a block.  A pool is (num_blocks, hkv) pieces of 9 * head_dim bytes, one per block and KV head: the codes of
// its sixteen rows (head_dim / 2 bytes each), then sixteen rows of (scale, bias) pairs of the 16-bit type T, a pair for every 64
// elements of a row.  So all that one KV head of a 16-token page takes is contiguous (1152 or 2304 bytes): one bulk copy.
// An element is scale * code + bias with, in a group of 64,
//
//   bias = min,   scale = T((max - min) / 15)   (0 below 2^-100),   code = min(15, rint((x - bias) / scale)),   x - bias in fp32,
//
// so min itself is held exactly, and an element is off by half a scale, and by 15 half units in the last place of the scale.
// Word r * (head_dim / 64) + g of a row holds elements 64 g + 8 r .. + 7: a lane that takes consecutive words gets the same
// share of every group, which is what keeps the fragments of the attention kernels inside one group's scale.
// Element e of a word sits in nibble e / 2 + 4 (e % 2): shifted by 4 i and masked, a word gives elements 2 i and 2 i + 1 in
// its halves, two neighbours of a 16-bit row.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace msgl {

constexpr int kKv4Rows = 16;     // slots of a block
constexpr int kKv4Group = 64;    // elements that share a scale and a bias
__host__ __device__ constexpr int kv4_block_bytes(int hd) { return 9 * hd; }
__host__ __device__ constexpr int kv4_pairs_at(int hd) { return 8 * hd; }   // byte offset of the pairs in a block
// What is held lies within +-2^15 (so that scale * code + bias is finite in either type, whichever way the scale was rounded):
// larger numbers and infinities are stored as that, NaN as 0, and the status word says so.
constexpr float kKv4Max = 32768.f;
constexpr int kKv4Reported = 4;

template <typename T>
struct Pack2;
template <>
struct Pack2<__nv_bfloat16> {
  using V = __nv_bfloat162;
};
template <>
struct Pack2<__half> {
  using V = __half2;
};
template <typename T>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  using V = typename Pack2<T>::V;
  const V r = __hmax2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  using V = typename Pack2<T>::V;
  const V r = __hmin2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The f16 numbers off + n of nibble i of both halves of a word, and off.  (Ten bits of fraction: the nibble at bit 4, 4, 2 and 6.)
__host__ __device__ constexpr float nibble_off(int i) { return i < 2 ? 64.f : i == 2 ? 256.f : 16.f; }
__device__ __forceinline__ uint32_t nibble_f16(uint32_t w, int i) {
  return i == 0   ? (((w << 4) & 0x00f000f0u) | 0x54005400u)
         : i == 1 ? ((w & 0x00f000f0u) | 0x54005400u)
         : i == 2 ? (((w >> 6) & 0x003c003cu) | 0x5c005c00u)
                  : (((w >> 6) & 0x03c003c0u) | 0x4c004c00u);
}

// BYTES at an aligned address, four to a word.
template <int BYTES>
__device__ __forceinline__ void read_words(uint32_t (&r)[BYTES / 4], const unsigned char* at) {
  if constexpr (BYTES == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    r[0] = x.x;
    r[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(at)[i];
      r[4 * i] = x.x;
      r[4 * i + 1] = x.y;
      r[4 * i + 2] = x.z;
      r[4 * i + 3] = x.w;
    }
  }
}

__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// The eight elements of a word under an f16 pair, in order: scale * code + bias in f16, rounded once (half a unit: 2^-11 of an
// element from 2^-14 on, which is what block_power is for).
__device__ __forceinline__ uint4 kv4_values(uint32_t word, uint32_t pair) {
  const uint32_t scale = __byte_perm(pair, pair, 0x1010), bias = __byte_perm(pair, pair, 0x3232);
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t one = MmaOp<__half>::pack(1.f, 1.f), off = MmaOp<__half>::pack(-nibble_off(i), -nibble_off(i));
    v[i] = fma_f16x2(fma_f16x2(nibble_f16(word, i), one, off), scale, bias);         // (the inner one is exact)
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A row's power of two, from its largest magnitude (the bits of a T): what is divided by it is below 2^11.
__device__ __forceinline__ float row_power(__half, uint32_t top) {
  const float x = __half2float(__ushort_as_half(static_cast<unsigned short>(top)));
  return __uint_as_float((max(__float_as_uint(x) >> 23, 12u) - 10u) << 23);
}
__device__ __forceinline__ float row_power(__nv_bfloat16, uint32_t top) {
  return __uint_as_float((max(top >> 7, 12u) - 10u) << 23);
}
// 1 / power, exactly (its exponent field is 1 to 253).
__device__ __forceinline__ float power_inverse(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }

// Powers of two for keys and values.  Elements go to the products as f16 numbers, and the pool's (scales from 2^-100, numbers to 2^15) are
// more than f16 has.  So the keys of a head that go into one sum are divided by a power of two, and so are the values; one comes
// back in the scores' scale, the other with the output.  Let t be the largest of their biases' magnitudes and 16 scales: elements are below
// 2 t, and the power brings t to [2^13, 2^14).  An element keeps f16's eleven bits down to 2^-27 of the largest one, and below that is
// held to 2^-38 of it.  At least 2^-95, so that sums over it stay finite; 1 where there is nothing.
// (Largest scales in the low halves and biases' magnitudes in the high ones: such bits are ordered as the numbers are.)
__device__ __forceinline__ uint32_t pair_tops(uint32_t tops, uint32_t pair) { return __vmaxu2(tops, pair & 0x7fff7fffu); }
// t, as the bits of a float.
template <typename T>
__device__ __forceinline__ uint32_t largest(uint32_t tops) {
  const float2 x = unpack_pair(T{}, tops);
  return __float_as_uint(fmaxf(16.f * x.x, x.y));
}
__device__ __forceinline__ float range_power(uint32_t top) {
  return top == 0u ? 1.f : __uint_as_float((min(max(top >> 23, 45u), 254u) - 13u) << 23);
}
// The largest t of K and of V over keys [t_lo, t_hi) of a sequence, of what this warp's threads look at (`thread` of THREADS that share the
// range): the pairs of a block of a head are 8 G words of 16 bytes in K and V together, one a thread.  block_of: a key's block in the pool.
template <typename T, int HD, int THREADS, typename BlockOf>
__device__ __forceinline__ uint2 pair_range(const unsigned char* k_pool, const unsigned char* v_pool, int hkv, int h, int t_lo, int t_hi,
                                            int64_t num_blocks, int thread, BlockOf block_of) {
  constexpr int G = HD / kKv4Group, UNITS = 8 * G, FLY = 4;
  constexpr int STEP = THREADS / UNITS * kKv4Rows;
  const int part = thread % (UNITS / 2);             // of 4 / G rows
  const bool is_v = thread % UNITS >= UNITS / 2;
  const unsigned char* const from = (is_v ? v_pool : k_pool) + static_cast<int64_t>(h) * kv4_block_bytes(HD) + kv4_pairs_at(HD) + part * 16;
  const int t_end = t_hi - part * 4 / G;             // its first row is a key below this
  uint32_t tops = 0u;
#pragma unroll 1
  for (int t0 = t_lo + thread / UNITS * kKv4Rows; t0 < t_hi; t0 += FLY * STEP) {
    int64_t block[FLY];
    uint4 x[FLY];
#pragma unroll
    for (int f = 0; f < FLY; ++f) block[f] = t0 + f * STEP < t_end ? block_of(t0 + f * STEP) : -1;
#pragma unroll
    for (int f = 0; f < FLY; ++f)
      x[f] = block[f] >= 0 && block[f] < num_blocks ? __ldg(reinterpret_cast<const uint4*>(from + block[f] * hkv * kv4_block_bytes(HD)))
                                                     : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int f = 0; f < FLY; ++f) {
      if (G == 2 && t0 + f * STEP + 1 >= t_end) x[f].z = x[f].w = 0u;      // (its second row)
      tops = pair_tops(pair_tops(pair_tops(pair_tops(tops, x[f].x), x[f].y), x[f].z), x[f].w);
    }
  }
  const uint32_t top = largest<T>(tops);
  return make_uint2(__reduce_max_sync(0xffffffffu, is_v ? 0u : top), __reduce_max_sync(0xffffffffu, is_v ? top : 0u));
}
// The largest weight of a row is put 2^7 above 1 (f16 ends at 2^16, and it may grow by 2^8 before it is put there again): a weight then has
// all its bits down to 2^-21 of the largest, where the value under it may be that much larger than the others.
constexpr float kWeightRoom = 7.f;
// A pair in f16, times a power of two.
template <typename T>
__device__ __forceinline__ uint32_t f16_pair(T, uint32_t pair, float by) {
  const float2 x = unpack_pair(T{}, pair);
  return MmaOp<__half>::pack(x.x * by, x.y * by);
}

// Codes of the 2 W elements that a lane holds of a group of 64, LANES = 32 / W lanes of `mask` together, and the group's pair
// (scale in the low half).  Element e comes back in nibble e / 2 + 4 (e % 2) of the result (W = 2: of its four lowest
// nibbles of each half, to be shifted by 8 for the upper half of a word).
// The quotient is an approximate one, corrected once by its exact remainder (Markstein), which makes it right at halves: x - bias and
// scale are short numbers whose quotient is often half-way between two codes, where a unit in the last place decides.
template <typename T, int W>
__device__ __forceinline__ uint32_t kv4_quantise(uint32_t (&x)[W], uint32_t mask, uint32_t& pair, int* status) {
  constexpr int LANES = 32 / W;
  float lo, hi;
#pragma unroll 1
  for (int again = 0;; ++again) {
    uint32_t mx = x[0], mn = x[0];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      mx = max2_nan<T>(mx, x[w]);
      mn = min2_nan<T>(mn, x[w]);
    }
    // (max, -min) in one word: one exchange for both
    uint32_t ends = max2_nan<T>(__byte_perm(mx, mn ^ 0x80008000u, 0x5410), __byte_perm(mx, mn ^ 0x80008000u, 0x7632));
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) ends = max2_nan<T>(ends, __shfl_xor_sync(mask, ends, o));
    const float2 e = unpack_pair(T{}, ends);
    hi = e.x;
    lo = -e.y;
    if ((fabsf(hi) <= kKv4Max && fabsf(lo) <= kKv4Max) || again) break;
    if (status) atomicOr(status, kKv4Reported);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      float2 v = unpack_pair(T{}, x[w]);
      v.x = v.x != v.x ? 0.f : fminf(fmaxf(v.x, -kKv4Max), kKv4Max);
      v.y = v.y != v.y ? 0.f : fminf(fmaxf(v.y, -kKv4Max), kKv4Max);
      x[w] = MmaOp<T>::pack(v.x, v.y);
    }
  }
  const float range = hi - lo;
  float fifteenth = range * (1.f / 15.f);
  fifteenth = fmaf(fmaf(-15.f, fifteenth, range), 1.f / 15.f, fifteenth);
  const T s16 = MmaOp<T>::from_float(fifteenth);
  const float scale = to_f32(s16);
  const bool flat = !(scale >= 7.888609052210118e-31f);   // 2^-100
  pair = MmaOp<T>::pack(flat ? 0.f : scale, lo);
  const float inv = flat ? 0.f : rcp_approx(scale);
  const uint64_t lo2 = pack_f32x2(-lo, -lo), inv2 = pack_f32x2(inv, inv), scale2 = pack_f32x2(-scale, -scale);
  const uint64_t magic = pack_f32x2(12582912.f, 12582912.f);     // 1.5 * 2^23: the sum's lowest bits are the rounded number
  // (a quotient is over 15.5 only where the scale was rounded down by more than 1/32, i.e. is subnormal)
  const bool clamp = std::is_same<T, __half>::value && scale < 6.103515625e-5f;
  uint32_t out = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float2 v = unpack_pair(T{}, x[w]);
    const uint64_t a = add_f32x2(pack_f32x2(v.x, v.y), lo2);
    uint64_t q = mul_f32x2(a, inv2);
    q = fma_f32x2(fma_f32x2(q, scale2, a), inv2, q);
    float q0, q1;
    if (clamp) {
      unpack_f32x2(q, q0, q1);
      q = pack_f32x2(fminf(q0, 15.f), fminf(q1, 15.f));
    }
    unpack_f32x2(add_f32x2(q, magic), q0, q1);
    out += __byte_perm(__float_as_uint(q0), __float_as_uint(q1), 0x5410) << (4 * w);
  }
  return out;
}

// ---------------------------------------------------------------- rows into the pool
// Token of a row (token * heads + head) without a division: the high half of a product with ceil(2^32 / heads) is it or one more.
__host__ __device__ __forceinline__ uint32_t row_reciprocal(uint32_t heads) {
  return heads == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + heads - 1) / heads);
}
__device__ __forceinline__ uint32_t token_of(uint32_t row, uint32_t heads, uint32_t recip) {
  if (recip == 0u) return row;
  const uint32_t t = __umulhi(row, recip);
  return t * heads > row ? t - 1 : t;
}

// Eight lanes a group, sixteen bytes of K and as many of V a lane: one exchange of (max, -min) over eight lanes, and K and V of a row
// under one look-up of its slot.  What bounds it is instruction issue (a quotient and a rounding for every element): 49152 tokens of
// 8 heads of 128 stored and read back, two launches, 113 to 115 us, 4.7 TB/s, 61 of them storing (with an exchange for each end and one
// quotient at a time 143); 24 tokens 8.6.
struct Kv4StoreParams {
  unsigned char *k_pool, *v_pool;
  const void *k, *v;          // (n, hkv, head_dim), dense heads
  const int32_t* slots;
  int64_t k_stride, v_stride; // elements between tokens
  int64_t num_slots;
  int n, hkv;
  uint32_t hkv_recip;         // see token_of
  int wide;                   // rows are 16-byte aligned
  int* status;
};

template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_store_kernel(Kv4StoreParams p) {
  constexpr int CH = HD / 8, G = HD / kKv4Group;
  grid_dependency_wait();
  grid_dependency_launch();
  const int32_t* slots = after_wait(p.slots);
  const T* k = after_wait(static_cast<const T*>(p.k));
  const T* v = after_wait(static_cast<const T*>(p.v));
  const int lane = threadIdx.x & 31;
  const uint32_t mask = 0xffu << (lane & 24);       // the eight lanes of a group
  constexpr uint32_t PER = 256 / CH;                // rows of a CTA at a time
  const uint32_t rows = static_cast<uint32_t>(p.n) * p.hkv;
  const int c = threadIdx.x % CH;                   // elements 8 c .. 8 c + 7
  for (uint32_t row = blockIdx.x * PER + threadIdx.x / CH; row < rows; row += gridDim.x * PER) {
    const uint32_t t = token_of(row, p.hkv, p.hkv_recip), h = row - t * p.hkv;
    const int slot = slots[t];
    if (slot < 0 || slot >= p.num_slots) {
      if (p.status) atomicOr(p.status, 2);
      continue;
    }
    const T* ks = k + t * p.k_stride + h * HD + c * 8;
    const T* vs = v + t * p.v_stride + h * HD + c * 8;
    uint32_t x[2][4];
    if (p.wide) {
      *reinterpret_cast<uint4*>(x[0]) = *reinterpret_cast<const uint4*>(ks);
      *reinterpret_cast<uint4*>(x[1]) = *reinterpret_cast<const uint4*>(vs);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        reinterpret_cast<uint2*>(x[0])[j] = reinterpret_cast<const uint2*>(ks)[j];
        reinterpret_cast<uint2*>(x[1])[j] = reinterpret_cast<const uint2*>(vs)[j];
      }
    }
    const int64_t block = (static_cast<int64_t>(slot / kKv4Rows) * p.hkv + h) * kv4_block_bytes(HD);
    const int r = slot % kKv4Rows, g = c / 8;
    const int64_t code_at = block + r * (HD / 2) + ((c % 8) * G + g) * 4;
    const int64_t pair_at = block + kv4_pairs_at(HD) + (r * G + g) * 4;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unsigned char* pool = j == 0 ? p.k_pool : p.v_pool;
      uint32_t pair;
      const uint32_t word = kv4_quantise<T, 4>(x[j], mask, pair, p.status);
      *reinterpret_cast<uint32_t*>(pool + code_at) = word;
      if (c % 8 == 0) *reinterpret_cast<uint32_t*>(pool + pair_at) = pair;
    }
  }
}

// ---------------------------------------------------------------- rows out of the pool
// A word and its pair a lane, of two rows at once, eight elements in order, rounded once from fp32.  Bound by memory: 52272 tokens of 8
// heads of 128 53 us, 5.2 TB/s (a row at a time 57).
struct Kv4LoadParams {
  const unsigned char *k_pool, *v_pool;
  void *k, *v;                // (n, hkv, head_dim), contiguous
  const int32_t* slots;
  int64_t num_slots;
  int n, hkv;
  uint32_t hkv_recip;
  int* status;
};

template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_load_kernel(Kv4LoadParams p) {
  constexpr int CH = HD / 8, G = HD / kKv4Group;
  grid_dependency_wait();
  grid_dependency_launch();
  const int32_t* slots = after_wait(p.slots);
  const unsigned char* pools[2] = {after_wait(p.k_pool), after_wait(p.v_pool)};
  constexpr uint32_t PER = 256 / CH;
  constexpr int RU = 2;                             // rows in flight
  const uint32_t rows = static_cast<uint32_t>(p.n) * p.hkv;
  const int c = threadIdx.x % CH, g = c / 8;
  for (uint32_t row0 = blockIdx.x * PER + threadIdx.x / CH; row0 < rows; row0 += gridDim.x * PER * RU) {
    uint32_t word[RU][2], pair[RU][2];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const uint32_t row = row0 + u * gridDim.x * PER;
      const uint32_t t = token_of(row, p.hkv, p.hkv_recip), h = row - t * p.hkv;
      const int slot = row < rows ? __ldg(slots + t) : 0;
      const bool ok = row < rows && slot >= 0 && slot < p.num_slots;
      if (!ok && row < rows && p.status) atomicOr(p.status, 2);
      const int64_t block = (static_cast<int64_t>(slot / kKv4Rows) * p.hkv + h) * kv4_block_bytes(HD);
      const int r = slot % kKv4Rows;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        word[u][j] = ok ? __ldg(reinterpret_cast<const uint32_t*>(pools[j] + block + r * (HD / 2) + ((c % 8) * G + g) * 4)) : 0u;
        pair[u][j] = ok ? __ldg(reinterpret_cast<const uint32_t*>(pools[j] + block + kv4_pairs_at(HD) + (r * G + g) * 4)) : 0u;
      }
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const uint32_t row = row0 + u * gridDim.x * PER;
      if (row >= rows) break;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 sb = unpack_pair(T{}, pair[u][j]);
        uint4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t n = word[u][j] >> (4 * e);
          reinterpret_cast<uint32_t*>(&o)[e] = MmaOp<T>::pack(fmaf(static_cast<float>(n & 15u), sb.x, sb.y),
                                                              fmaf(static_cast<float>(n >> 16 & 15u), sb.x, sb.y));
        }
        reinterpret_cast<uint4*>(j == 0 ? p.k : p.v)[static_cast<int64_t>(row) * CH + c] = o;
      }
    }
  }
}

// ---------------------------------------------------------------- pages laid out for the pairs of CTAs
// A long prefill reads a key once for every 256 query rows, and to expand its codes each time is what bounds the kernel that does
// (one CTA; 4096 tokens over 16384 1425 us when that was measured).  Expanded once into f16 pages, one per entry of the index list and
// in its order, they come by TMA and pairs of CTAs share them.  A sequence's keys and values of a head are divided by powers of two
// (range_power), which a kernel in front finds.  q goes with them, as f16 over a power of two per row (bf16 only).
// Bound by memory: 2.6 bytes an element of the pool, 4 of q; 20480 tokens of 8 heads of 128 and 4096 queries of 32 heads 34 us, 5.2
// TB/s, in front of an attention of 990 (with 116 registers and two CTAs per SM 44).
struct Kv4ExpandParams {
  const unsigned char *k_pool, *v_pool;
  const int32_t* page_indices;
  __half *k_rows, *v_rows;      // (total_pages * page_size, hkv, head_dim)
  int32_t* pages;               // (total_pages): 0, 1, ...
  uint32_t* tops;               // (batch, hkv, 2, kRangeParts): the largest t of K and of V in parts of a sequence
  const int32_t *page_indptr, *kv_lens, *prefix_lens, *qo_indptr;
  int batch, window, is_cross;
  int parts;                    // CTAs of a sequence and head in kv4_range_kernel: a power of two up to kRangeParts
  const void* q;                // (q_rows, head_dim), or null
  __half* q_rows;
  float* q_power;
  int total_pages, page_blocks, hkv, num_blocks;
  int64_t num_q_rows;
  int* status;
};

constexpr int kRangeParts = 32;
// What a sequence's keys (is_v: values) of a head are divided by, for a warp.
__device__ __forceinline__ float sequence_power(const uint32_t* tops, int b, int hkv, int h, int is_v, int lane) {
  return range_power(__reduce_max_sync(0xffffffffu, __ldg(tops + ((static_cast<int64_t>(b) * hkv + h) * 2 + is_v) * kRangeParts + lane)));
}

// A CTA for each part of each sequence and head: the keys from the first that a row's window can reach (and the tile of 128 that it is
// in) to the last.  A ninth of the pool is read; 20480 tokens of 8 heads 6 us.
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_range_kernel(const Kv4ExpandParams p) {
  __shared__ uint2 s_top[8];
  grid_dependency_wait();
  grid_dependency_launch();
  const int32_t* const ids = after_wait(p.page_indices);
  const int32_t* const indptr = after_wait(p.page_indptr);
  const int32_t* const lens = after_wait(p.kv_lens);
  const int32_t* const prefixes = after_wait(p.prefix_lens);
  const int part = blockIdx.x % p.parts, h = blockIdx.x / p.parts % p.hkv, b = blockIdx.x / p.parts / p.hkv;
  const int page_size = p.page_blocks * kKv4Rows;
  const int begin = __ldg(indptr + b);
  const int64_t cap = static_cast<int64_t>(max(__ldg(indptr + b + 1) - begin, 0)) * page_size;
  const int len = static_cast<int>(min(static_cast<int64_t>(max(__ldg(lens + b), 0)), cap));
  const int lo = p.window > 0 ? max(0, __ldg(prefixes + b) - p.window + 1) / 128 * 128 : 0;
  const int per = (max(len - lo, 0) / kKv4Rows / p.parts + 1) * kKv4Rows;        // keys of a part
  const int64_t from = lo + static_cast<int64_t>(part) * per;
  uint2 top = make_uint2(0u, 0u);
  if (from < len)
    top = pair_range<T, HD, 256>(after_wait(p.k_pool), after_wait(p.v_pool), p.hkv, h, static_cast<int>(from),
                                 static_cast<int>(min(from + per, static_cast<int64_t>(len))), p.num_blocks, threadIdx.x, [&](int t) -> int64_t {
                                   const int page = t / page_size, at = begin + page;
                                   if (at < 0 || at >= p.total_pages) return -1;
                                   return static_cast<int64_t>(__ldg(ids + at)) * p.page_blocks + (t - page * page_size) / kKv4Rows;
                                 });
  if (threadIdx.x % 32 == 0) s_top[threadIdx.x / 32] = top;
  __syncthreads();
  // (with fewer CTAs than places, all its places hold the same)
  const int is_v = threadIdx.x / kRangeParts, place = threadIdx.x % kRangeParts;
  if (is_v < 2 && place % p.parts == part) {
    uint32_t most = 0u;
#pragma unroll
    for (int w = 0; w < 8; ++w) most = max(most, is_v == 0 ? s_top[w].x : s_top[w].y);
    p.tops[((static_cast<int64_t>(b) * p.hkv + h) * 2 + is_v) * kRangeParts + place] = most;
  }
}

// The sequence that `page` (an entry of the index list) belongs to: a search by the warp in the row pointers, for the last that is
// at most `page`.
__device__ __forceinline__ int sequence_of_page(const int32_t* indptr, int batch, int page, int lane) {
  int first = 0, n = batch;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lane * step;
    const uint32_t in = __ballot_sync(0xffffffffu, at < n && __ldg(indptr + first + min(at, n - 1)) <= page);
    const int k = in == 0u ? 0 : 31 - __clz(in);
    first += k * step;
    n = min(step, n - k * step);
  }
  return first;
}

template <typename T, int HD>
__global__ void __launch_bounds__(256, 4) kv4_expand_kernel(const Kv4ExpandParams p) {
  constexpr int CH = HD / 8, G = HD / kKv4Group, RPP = 32 / CH;      // chunks of a row; rows a pass of a warp
  grid_dependency_wait();
  grid_dependency_launch();
  const int32_t* ids = after_wait(p.page_indices);
  const int32_t* const indptr = after_wait(p.page_indptr);
  const int32_t* const lens = after_wait(p.kv_lens);
  const int32_t* const prefixes = after_wait(p.prefix_lens);
  const int32_t* const new_tokens = after_wait(p.qo_indptr);
  const uint32_t* const tops = after_wait(p.tops);
  const unsigned char* pools[2] = {after_wait(p.k_pool), after_wait(p.v_pool)};
  const T* q = after_wait(static_cast<const T*>(p.q));
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * 8, first = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int c = lane % CH, rsub = lane / CH;
  const int word_at = ((c % 8) * G + c / 8) * 4, pair_at = kv4_pairs_at(HD) + c / 8 * 4;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < p.total_pages; i += gridDim.x * 256ll) p.pages[i] = static_cast<int>(i);
  // a warp a block of a head, K and V
  const int64_t blocks = static_cast<int64_t>(p.total_pages) * p.page_blocks;
  for (int64_t i = first; i < blocks * p.hkv; i += warps) {
    const int64_t b = i / p.hkv;
    const int h = static_cast<int>(i - b * p.hkv);
    const int page = p.page_blocks == 1 ? static_cast<int>(b) : static_cast<int>(b / p.page_blocks);
    const int64_t block = static_cast<int64_t>(__ldg(ids + page)) * p.page_blocks + (b - static_cast<int64_t>(page) * p.page_blocks);
    const bool ok = block >= 0 && block < p.num_blocks;
    const int seq = sequence_of_page(indptr, p.batch, page, lane);
    const int64_t t = b * kKv4Rows - static_cast<int64_t>(__ldg(indptr + seq)) * p.page_blocks * kKv4Rows;     // its first token
    const int len = __ldg(lens + seq);
    if (t < 0 || t >= len) continue;              // an entry that no sequence has a token in: not read, and not reported
    if (!ok && lane == 0 && p.status) {           // reported where a row sees it
      const int prefix = __ldg(prefixes + seq), fresh = __ldg(new_tokens + seq + 1) - __ldg(new_tokens + seq);
      if ((p.is_cross || t < static_cast<int64_t>(prefix) + fresh) && (p.window == 0 || t + kKv4Rows > static_cast<int64_t>(prefix) - p.window + 1))
        atomicOr(p.status, 2);
    }
    const int64_t at = ((ok ? block : 0) * p.hkv + h) * kv4_block_bytes(HD);
    const float inverse[2] = {power_inverse(sequence_power(tops, seq, p.hkv, h, 0, lane)),
                              power_inverse(sequence_power(tops, seq, p.hkv, h, 1, lane))};
#pragma unroll (HD == 128 ? 2 : 1)
    for (int j = 0; j < 2; ++j) {
      const unsigned char* src = (j == 0 ? pools[0] : pools[1]) + at;
      const float by = j == 0 ? inverse[0] : inverse[1];
      uint32_t word[kKv4Rows / RPP], pair[kKv4Rows / RPP];
#pragma unroll
      for (int k = 0; k < kKv4Rows / RPP; ++k) {
        const int r = k * RPP + rsub;
        word[k] = ok ? __ldg(reinterpret_cast<const uint32_t*>(src + r * (HD / 2) + word_at)) : 0u;
        pair[k] = ok ? __ldg(reinterpret_cast<const uint32_t*>(src + pair_at + r * (G * 4))) : 0u;
      }
      __half* const dst = (j == 0 ? p.k_rows : p.v_rows) + (b * kKv4Rows * p.hkv + h) * HD + c * 8;
#pragma unroll
      for (int k = 0; k < kKv4Rows / RPP; ++k)
        *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(k * RPP + rsub) * p.hkv * HD) =
            kv4_values(word[k], f16_pair(T{}, pair[k], by));
    }
  }
  if (q == nullptr) return;
  const uint32_t mask = CH == 32 ? 0xffffffffu : (lane & 16) ? 0xffff0000u : 0x0000ffffu;
  for (int64_t row = first * RPP + rsub; row < p.num_q_rows; row += warps * RPP) {
    uint4 x = *reinterpret_cast<const uint4*>(q + row * HD + c * 8);
    uint32_t* const w = reinterpret_cast<uint32_t*>(&x);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, max(w[e] >> 16 & 0x7fffu, w[e] & 0x7fffu));
#pragma unroll
    for (int o = 1; o < CH; o <<= 1) top = max(top, __shfl_xor_sync(mask, top, o));
    const float power = row_power(T{}, top), inv = power_inverse(power);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_pair(T{}, w[e]);
      w[e] = MmaOp<__half>::pack(f.x * inv, f.y * inv);
    }
    *reinterpret_cast<uint4*>(p.q_rows + row * HD + c * 8) = x;
    if (c == 0) p.q_power[row] = power;
  }
}

}  // namespace msgl
