// Norm, rotation and append in one pass for the 4-bit pool (kv4.cuh): per-head RMSNorm of q and k, rotary embedding of both,
// q to a new tensor, k and v quantised into the pool.  Every row is read once and written once.
//
// y = x * rsqrt(mean(x^2) + eps) * w in fp32, rounded to the 16-bit type (the array that the layer's norm gives); pairs
// (i, i + rd/2) rotated by position * base^(-2i/rd), rounded once more; what is quantised is that rounded key, the one a
// 16-bit pool would hold.  Where a rounding falls the other way a code can, and an element is off by a whole step of its
// group, so the chain in front of the roundings is that of separate fp32 operations, over sines and
// cosines that are those of 64 bits rounded once: the angle is kept in quarter turns, position times frequency in 64 bits, exact to 2^-37 of one
// at 10^5 tokens, and what is left of it within an eighth of a turn goes into Taylor's polynomials to the 13th power.  (Products fused with the sum
// behind them turn one rounding in 10^5 the other way.)
//
// A work item is a few rows of one token and one kind (q, k or v), one after the other, the next on its way: angles and
// weights are the item's, and the code is short (with four rows unrolled the kernel waited for instructions as much as for
// anything).  head_dim / 8 lanes take it; lane l holds elements
// 4 l .. 4 l + 3 of the lower half of a row and as many half a row further on, so that with rotary_dim = head_dim a pair is in
// one lane, and a group of 64 is in sixteen lanes.
//
// What bounds it is instruction issue, some 250 instructions a row that is quantised: 6000 tokens of 16 + 2 x 4 heads of 256, and the
// read back behind it, 51.6 us, 3.2 TB/s (one element at a time and four rows an item unrolled: 74; squares through shared memory 53).
#pragma once

#include "kv4.cuh"

namespace msgl {

struct Kv4ProjectParams {
  const void *q, *k, *v;
  void* q_out;               // (n, hq, head_dim), contiguous
  const void *q_weight, *k_weight;
  const int32_t *positions, *slots;
  unsigned char *k_pool, *v_pool;
  int n, hq, hkv, rotary_dim;
  int item_rows;             // rows of an item at most
  int64_t q_stride, k_stride, v_stride;
  int64_t num_slots;
  double log2_base;
  float eps;
  float minus_zero;          // -0, which the compiler does not know: see product
  int* status;
};
__host__ __device__ constexpr int kv4_project_lanes(int hd) { return hd / 8; }

// Sine and cosine of pos * freq quarter turns (below 2^51 of them).
__device__ __forceinline__ void sine_cosine(double pos, double freq, float& sine, float& cosine) {
  const double magic = 6755399441055744.;                  // 1.5 * 2^52: the sum's lowest bits are the rounded number
  const double whole = fma(pos, freq, magic);
  const double z = fma(pos, freq, magic - whole) * 1.5707963267948966, y = z * z;      // |z| <= pi / 4
  double s = fma(y, 1. / 6227020800., -1. / 39916800.), c = fma(y, 1. / 479001600., -1. / 3628800.);
  s = fma(y, s, 1. / 362880.);
  c = fma(y, c, 1. / 40320.);
  s = fma(y, s, -1. / 5040.);
  c = fma(y, c, -1. / 720.);
  s = fma(y, s, 1. / 120.);
  c = fma(y, c, 1. / 24.);
  s = fma(y, s, -1. / 6.);
  c = fma(y, c, -1. / 2.);
  const float s1 = static_cast<float>(fma(y * z, s, z)), c1 = static_cast<float>(fma(y, c, 1.));
  const int k = __double2loint(whole);                     // quarter turns, modulo 4
  sine = k & 1 ? c1 : s1;
  cosine = k & 1 ? s1 : c1;
  if (k & 2) sine = -sine;
  if ((k + 1) & 2) cosine = -cosine;
}

template <typename T, int HD>
__global__ void __launch_bounds__(256, 4) kv4_project_kernel(const Kv4ProjectParams p) {
  constexpr int LANES = kv4_project_lanes(HD), G = HD / kKv4Group;
  const int R = p.item_rows;
  __shared__ __align__(16) float s_weight[2][HD];
  const int lane = threadIdx.x & 31;
  const int hl = lane & (LANES - 1);
  // A product that stays one: mul.rn.f32x2 and the add behind it come out of the compiler as one operation.
  const uint64_t nothing = pack_f32x2(p.minus_zero, p.minus_zero);
  auto product = [&](uint64_t a, uint64_t b) -> uint64_t { return fma_f32x2(a, b, nothing); };
  const uint32_t hmask = LANES == 32 ? 0xffffffffu : (lane & 16) ? 0xffff0000u : 0x0000ffffu;
  const uint32_t gmask = (lane & 16) ? 0xffff0000u : 0x0000ffffu;     // the sixteen lanes of a group
  const int half = p.rotary_dim >> 1;
  const bool in_lane = p.rotary_dim == HD;
  const int xm = in_lane ? 0 : half / 4;             // pairs inside the lower half of the row: the partner is lane ^ xm
  const bool rot_lane = in_lane || hl < 2 * xm;
  const int f0 = in_lane ? 4 * hl : 4 * (hl & (xm - 1));
  double freq[4];                                    // quarter turns per token
#pragma unroll
  for (int e = 0; e < 4; ++e) freq[e] = exp2(-p.log2_base * static_cast<double>(f0 + e) / half) * 0.63661977236758134;
  grid_dependency_wait();
  grid_dependency_launch();
  const T* const q = after_wait(static_cast<const T*>(p.q));
  const T* const k = after_wait(static_cast<const T*>(p.k));
  const T* const v = after_wait(static_cast<const T*>(p.v));
  const int32_t* const positions = after_wait(p.positions);
  const int32_t* const slots = after_wait(p.slots);
  for (int e = threadIdx.x; e < 2 * HD; e += 256) {
    const T* w = static_cast<const T*>(e < HD ? p.q_weight : p.k_weight);
    if (w != nullptr) s_weight[e / HD][e % HD] = to_f32(w[e % HD]);
  }
  __syncthreads();
  const uint32_t gq = (p.hq + R - 1) / R, gk = (p.hkv + R - 1) / R;
  const uint32_t groups = gq + 2 * gk;
  const uint32_t total = static_cast<uint32_t>(p.n) * groups;
  for (uint32_t item = (blockIdx.x * blockDim.x + threadIdx.x) / LANES; item < total; item += gridDim.x * (256 / LANES)) {
    const uint32_t tok = item / groups;
    const uint32_t g = item - tok * groups;
    const bool is_q = g < gq, is_v = g >= gq + gk;
    const int h0 = static_cast<int>(is_q ? g : is_v ? g - gq - gk : g - gq) * R;
    const int cnt = min(R, (is_q ? p.hq : p.hkv) - h0);
    const T* src = (is_q ? q + tok * p.q_stride : is_v ? v + tok * p.v_stride : k + tok * p.k_stride) + h0 * HD;
    int slot = 0;
    if (!is_q) {
      slot = slots[tok];
      if (slot < 0 || slot >= p.num_slots) {
        if (p.status) atomicOr(p.status, 2);
        continue;
      }
    }
    uint64_t cs[2], sn[2], sm[2];       // cos, sin; what the other member of a pair is multiplied with in the lower half
    const bool norm = (is_q ? p.q_weight : p.k_weight) != nullptr;
    const float* weight = s_weight[is_q ? 0 : 1];
    uint2 lo = reinterpret_cast<const uint2*>(src)[hl], hi = reinterpret_cast<const uint2*>(src)[LANES + hl];
    if (!is_v) {
      const double pos = static_cast<double>(positions[tok]);
      float c4[4], s4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) sine_cosine(pos, freq[e], s4[e], c4[e]);
      const float sign = in_lane || hl < xm ? -1.f : 1.f;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        cs[w] = pack_f32x2(c4[2 * w], c4[2 * w + 1]);
        sn[w] = pack_f32x2(s4[2 * w], s4[2 * w + 1]);
        sm[w] = pack_f32x2(sign * s4[2 * w], sign * s4[2 * w + 1]);
      }
    }
#pragma unroll 1
    for (int r = 0; r < cnt; ++r) {
      uint2 lo1 = lo, hi1 = hi;
      if (r + 1 < cnt) {
        lo1 = reinterpret_cast<const uint2*>(src + (r + 1) * HD)[hl];
        hi1 = reinterpret_cast<const uint2*>(src + (r + 1) * HD)[LANES + hl];
      }
      if (!is_v) {
        auto open = [](uint32_t x) {
          const float2 f = unpack_pair(T{}, x);
          return pack_f32x2(f.x, f.y);
        };
        auto close = [](uint64_t x) {
          float f0, f1;
          unpack_f32x2(x, f0, f1);
          return MmaOp<T>::pack(f0, f1);
        };
        uint64_t a[2] = {open(lo.x), open(lo.y)}, b[2] = {open(hi.x), open(hi.y)};
        if (norm) {
          // sum of the squares: this lane's eight elements, then the lanes'
          float ss;
          if constexpr (LANES == 32) {
            float x0, x1, x2, x3;
            unpack_f32x2(add_f32x2(product(a[0], a[0]), product(b[0], b[0])), x0, x1);
            unpack_f32x2(add_f32x2(product(a[1], a[1]), product(b[1], b[1])), x2, x3);
            ss = __fadd_rn(__fadd_rn(__fadd_rn(x0, x1), x2), x3);
          } else {
            auto four = [&](const uint64_t (&x)[2]) -> float {
              float x0, x1, x2, x3;
              unpack_f32x2(product(x[0], x[0]), x0, x1);
              unpack_f32x2(product(x[1], x[1]), x2, x3);
              return __fadd_rn(__fadd_rn(__fadd_rn(x0, x1), x2), x3);
            };
            ss = __fadd_rn(four(a), four(b));
          }
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(hmask, ss, o));
          const float inv = rsqrtf(ss * (1.f / HD) + p.eps);
          const uint64_t inv2 = pack_f32x2(inv, inv);
          const ulonglong2 wl = reinterpret_cast<const ulonglong2*>(weight)[hl], wh = reinterpret_cast<const ulonglong2*>(weight)[LANES + hl];
          a[0] = open(close(mul_f32x2(mul_f32x2(a[0], inv2), wl.x)));
          a[1] = open(close(mul_f32x2(mul_f32x2(a[1], inv2), wl.y)));
          b[0] = open(close(mul_f32x2(mul_f32x2(b[0], inv2), wh.x)));
          b[1] = open(close(mul_f32x2(mul_f32x2(b[1], inv2), wh.y)));
        }
        if (in_lane) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint64_t x = a[w];
            a[w] = add_f32x2(product(x, cs[w]), product(b[w], sm[w]));
            b[w] = add_f32x2(product(b[w], cs[w]), product(x, sn[w]));
          }
        } else {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint64_t other = __shfl_xor_sync(hmask, static_cast<unsigned long long>(a[w]), xm);
            if (rot_lane) a[w] = add_f32x2(product(a[w], cs[w]), product(other, sm[w]));
          }
        }
        lo = make_uint2(close(a[0]), close(a[1]));
        hi = make_uint2(close(b[0]), close(b[1]));
      }
      if (is_q) {
        T* dst = static_cast<T*>(p.q_out) + (static_cast<int64_t>(tok) * p.hq + h0 + r) * HD;
        reinterpret_cast<uint2*>(dst)[hl] = lo;
        reinterpret_cast<uint2*>(dst)[LANES + hl] = hi;
      } else {
        // (lower half of the row: groups 0 .. G/2 - 1, lane l in group l / 16, word 8 g + (l % 16) / 2 in the order of the row;
        // an even lane writes the word of the lower half, its neighbour that of the upper half)
        const int row = slot % kKv4Rows;
        const int gw = hl / 16 + (hl & 1) * (G / 2), r8 = (hl & 15) >> 1;
        unsigned char* block = (is_v ? p.v_pool : p.k_pool) +
                               (static_cast<int64_t>(slot / kKv4Rows) * p.hkv + h0 + r) * kv4_block_bytes(HD);
        uint32_t xl[2] = {lo.x, lo.y}, xh[2] = {hi.x, hi.y};
        uint32_t pl, ph;
        const uint32_t cl = kv4_quantise<T, 2>(xl, gmask, pl, p.status) << (8 * (hl & 1));
        const uint32_t ch = kv4_quantise<T, 2>(xh, gmask, ph, p.status) << (8 * (hl & 1));
        // what the neighbour writes goes to it
        const uint32_t other = __shfl_xor_sync(gmask, (hl & 1) ? cl : ch, 1);
        *reinterpret_cast<uint32_t*>(block + row * (HD / 2) + (r8 * G + gw) * 4) = other | ((hl & 1) ? ch : cl);
        if ((hl & 15) < 2)
          *reinterpret_cast<uint32_t*>(block + kv4_pairs_at(HD) + (row * G + gw) * 4) = (hl & 1) ? ph : pl;
      }
      lo = lo1;
      hi = hi1;
    }
  }
}

}  // namespace msgl
