// Norm, rotation and append in one pass for the 4-bit pool (kv4.cuh): per-head RMSNorm of q and k, rotary embedding of both,
// q to a new tensor, k and v quantised into the pool.  Every row is read once and written once.
//
// y = x * rsqrt(mean(x^2) + eps) * w in fp32, rounded to the 16-bit type (the array that the layer's norm gives); pairs
// (i, i + rd/2) rotated by position * base^(-2i/rd), rounded once more; what is quantised is that rounded key, the one a
// 16-bit pool would hold.  Where a rounding falls the other way a code can, and an element is off by a whole step of its
// group, so the chain in front of the roundings is that of separate fp32 operations (no product is fused with a sum), and sine and cosine are good to a unit
// in the last place: the angle is kept in turns, position times a frequency of two floats, exact to 2^-33 turns at 10^5
// tokens (one float of frequency leaves an angle of 10^5 radians 6e-3 off).
//
// A work item is up to four rows of one token and one kind (q, k or v).  head_dim / 8 lanes take it; lane l holds elements
// 4 l .. 4 l + 3 of the lower half of a row and as many half a row further on, so that with rotary_dim = head_dim a pair is in
// one lane, and a group of 64 is in sixteen lanes.
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
  int64_t q_stride, k_stride, v_stride;
  int64_t num_slots;
  double log2_base;
  float eps;
  int* status;
};
constexpr int kKv4RowsPerItem = 4;
__host__ __device__ constexpr int kv4_project_lanes(int hd) { return hd / 8; }

template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_project_kernel(const Kv4ProjectParams p) {
  constexpr int LANES = kv4_project_lanes(HD), R = kKv4RowsPerItem, G = HD / kKv4Group;
  const int lane = threadIdx.x & 31;
  const int hl = lane & (LANES - 1);
  const uint32_t hmask = LANES == 32 ? 0xffffffffu : (lane & 16) ? 0xffff0000u : 0x0000ffffu;
  const uint32_t gmask = (lane & 16) ? 0xffff0000u : 0x0000ffffu;     // the sixteen lanes of a group
  const int half = p.rotary_dim >> 1;
  const bool in_lane = p.rotary_dim == HD;
  const int xm = in_lane ? 0 : half / 4;             // pairs inside the lower half of the row: the partner is lane ^ xm
  const bool rot_lane = in_lane || hl < 2 * xm;
  const int f0 = in_lane ? 4 * hl : 4 * (hl & (xm - 1));
  float f_hi[4], f_lo[4];                            // turns per token
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double f = exp2(-p.log2_base * static_cast<double>(f0 + e) / half) * 0.15915494309189535;
    f_hi[e] = static_cast<float>(f);
    f_lo[e] = static_cast<float>(f - f_hi[e]);
  }
  grid_dependency_wait();
  grid_dependency_launch();
  const T* const q = after_wait(static_cast<const T*>(p.q));
  const T* const k = after_wait(static_cast<const T*>(p.k));
  const T* const v = after_wait(static_cast<const T*>(p.v));
  const int32_t* const positions = after_wait(p.positions);
  const int32_t* const slots = after_wait(p.slots);
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
    uint2 lo[R], hi[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < cnt) {
        lo[r] = reinterpret_cast<const uint2*>(src + r * HD)[hl];
        hi[r] = reinterpret_cast<const uint2*>(src + r * HD)[LANES + hl];
      }
    }
    int slot = 0;
    if (!is_q) {
      slot = slots[tok];
      if (slot < 0 || slot >= p.num_slots) {
        if (p.status) atomicOr(p.status, 2);
        continue;
      }
    }
    if (!is_v) {
      const float pos = static_cast<float>(positions[tok]);
      float cs[4], sn[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float t = pos * f_hi[e];
        const float rest = fmaf(pos, f_lo[e], fmaf(pos, f_hi[e], -t));
        const float part = t - rintf(t), x = part + rest;              // turns, in [-1/2, 1/2]
        const float off = 6.2831854820251465f * (rest - (x - part));   // what the sum lost, in radians
        float s0, c0;
        sincospif(2.f * x, &s0, &c0);
        sn[e] = fmaf(off, c0, s0);
        cs[e] = fmaf(-off, s0, c0);
      }
      const T* wt = static_cast<const T*>(is_q ? p.q_weight : p.k_weight);
      uint2 wl = make_uint2(0u, 0u), wh = wl;
      if (wt != nullptr) {
        wl = reinterpret_cast<const uint2*>(wt)[hl];
        wh = reinterpret_cast<const uint2*>(wt)[LANES + hl];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= cnt) break;
        float a[4], b[4];
        auto open = [](const uint2& x, float (&f)[4]) {
          const float2 u = unpack_pair(T{}, x.x), w = unpack_pair(T{}, x.y);
          f[0] = u.x;
          f[1] = u.y;
          f[2] = w.x;
          f[3] = w.y;
        };
        auto close = [](const float (&f)[4]) { return make_uint2(MmaOp<T>::pack(f[0], f[1]), MmaOp<T>::pack(f[2], f[3])); };
        open(lo[r], a);
        open(hi[r], b);
        if (wt != nullptr) {
          // Sum of the squares, of elements 32 apart first and then of neighbours.  Lane l = 8 i + m holds elements 4 m .. 4 m + 3
          // of the row's i-th 32 in its lower half, and of the i-th 32 of its upper half.
          float t4[4];
          if constexpr (LANES == 32) {
            float u4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u4[e] = __fadd_rn(__fmul_rn(a[e], a[e]), __fmul_rn(b[e], b[e]));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              t4[e] = __shfl_sync(hmask, u4[e], hl & 7);
#pragma unroll
              for (int i = 1; i < 4; ++i) t4[e] = __fadd_rn(t4[e], __shfl_sync(hmask, u4[e], (hl & 7) + 8 * i));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = __fmul_rn(a[e], a[e]), y = __fmul_rn(b[e], b[e]);
              const float ox = __shfl_xor_sync(hmask, x, 8), oy = __shfl_xor_sync(hmask, y, 8);
              t4[e] = __fadd_rn(__fadd_rn(__fadd_rn(x, ox), hl & 8 ? oy : y), hl & 8 ? y : oy);
            }
          }
          float ss = __fadd_rn(__fadd_rn(t4[0], t4[1]), __fadd_rn(t4[2], t4[3]));
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(hmask, ss, o));
          const float inv = rsqrtf(ss * (1.f / HD) + p.eps);
          float x[4], y[4];
          open(wl, x);
          open(wh, y);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] = a[e] * inv * x[e];
            b[e] = b[e] * inv * y[e];
          }
          open(close(a), a);
          open(close(b), b);
        }
        if (in_lane) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = a[e];
            a[e] = __fsub_rn(__fmul_rn(x, cs[e]), __fmul_rn(b[e], sn[e]));
            b[e] = __fadd_rn(__fmul_rn(b[e], cs[e]), __fmul_rn(x, sn[e]));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float other = __shfl_xor_sync(hmask, a[e], xm);
            if (rot_lane) a[e] = __fadd_rn(__fmul_rn(a[e], cs[e]), __fmul_rn(other, hl >= xm ? sn[e] : -sn[e]));
          }
        }
        lo[r] = close(a);
        hi[r] = close(b);
      }
    }
    if (is_q) {
      T* dst = static_cast<T*>(p.q_out) + (static_cast<int64_t>(tok) * p.hq + h0) * HD;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < cnt) {
          reinterpret_cast<uint2*>(dst + r * HD)[hl] = lo[r];
          reinterpret_cast<uint2*>(dst + r * HD)[LANES + hl] = hi[r];
        }
      }
      continue;
    }
    const int row = slot % kKv4Rows;
    // (lower half of the row: groups 0 .. G/2 - 1, lane l in group l / 16, word 8 g + (l % 16) / 2 in the order of the row;
    // an even lane writes the word of the lower half, its neighbour that of the upper half)
    const int gl = hl / 16;
    const int gw = gl + (hl & 1) * (G / 2), r8 = (hl & 15) >> 1;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= cnt) break;
      unsigned char* block = (is_v ? p.v_pool : p.k_pool) +
                             (static_cast<int64_t>(slot / kKv4Rows) * p.hkv + h0 + r) * kv4_block_bytes(HD);
      uint32_t xl[2] = {lo[r].x, lo[r].y}, xh[2] = {hi[r].x, hi[r].y};
      uint32_t pl, ph;
      const uint32_t cl = kv4_quantise<T, 2>(xl, gmask, pl, p.status) << (8 * (hl & 1));
      const uint32_t ch = kv4_quantise<T, 2>(xh, gmask, ph, p.status) << (8 * (hl & 1));
      // what the neighbour writes goes to it
      const uint32_t other = __shfl_xor_sync(gmask, (hl & 1) ? cl : ch, 1);
      *reinterpret_cast<uint32_t*>(block + row * (HD / 2) + (r8 * G + gw) * 4) = other | ((hl & 1) ? ch : cl);
      if ((hl & 15) < 2)
        *reinterpret_cast<uint32_t*>(block + kv4_pairs_at(HD) + (row * G + gw) * 4) = (hl & 1) ? ph : pl;
    }
  }
}

}  // namespace msgl
