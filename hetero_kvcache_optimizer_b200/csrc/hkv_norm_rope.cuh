// Norm of query and key heads with the position rotation, in one pass.
// Included by hetero_kv.cu.
//
// Per row x (one head of one token, D = 128), in fp32 with one rounding at the end:
//   y = x * rsqrt(mean(x^2) + eps) * w          (only with a norm weight w)
//   (a, b) -> (a c - b s, b c + a s)            for the first `rot` dims of y
// where pair i is dims (i, i + rot/2), or (2i, 2i + 1) with `adjacent`, and
// (c, s) = (table[pos][i], table[pos][rot/2 + i]).
//
// Bound: HBM, each row read and written once (the table row of a token serves all
// of its heads). A half-warp holds a row (16 lanes x 8 values: one 16-byte load
// and store a lane), and a warp takes kHeads heads of ONE token, two rows at a
// time: cos and sin stay in registers for all of them, and all loads of the
// warp's rows are in flight before the first is used. A pair's other half is 8 k
// dims away when rot % 16 == 0, so it sits in the same register of another lane
// (one shuffle); other sizes read it from the row again (L1).
// The next launch is let in after this one's wait, so that it never runs beside
// a grid two launches back.
#pragma once
#include "hkv_common.cuh"

namespace hkv {

struct NormRopeParams {
  const void* x[2];        // q, k: [B][H][T][128]
  void* y[2];              // q_out, k_out (may be x)
  const void* w[2];        // norm weights [128] or NULL
  int w_dtype[2];
  int H[2];
  int64_t xs[2][3], ys[2][3];  // strides (b, h, t) in elements
  int vec[2];              // x, y rows 16-byte aligned
  const void* pos;         // int32 or int64 [B][T]
  int pos64;
  int64_t ps_b, ps_t;
  const float* table;      // [max_pos][rot]: cos | sin
  int64_t table_stride;    // elements
  int max_pos, rot;
  float eps;
  int B, T;
  int chunks[2];           // warps' head chunks per token of q and of k
};

constexpr int kNrThreads = 256;

// Half-split pairs whose halves are whole lanes apart | pairs of neighbours | any other half-split
enum { kNrLane = 0, kNrAdjacent = 1, kNrAny = 2 };

template <typename T>
__device__ __forceinline__ void nr_unpack(const uint4& r, float (&v)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T* h = reinterpret_cast<const T*>(&w[i]);
    v[2 * i] = to_f32(h[0]);
    v[2 * i + 1] = to_f32(h[1]);
  }
}

// Eight values from element `i` of a row: one 16-byte load, or eight 2-byte ones.
template <typename T>
__device__ __forceinline__ uint4 nr_load(const T* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * i;
    w[i] = (uint32_t)h[0] | ((uint32_t)h[1] << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// kHeads: heads of one token a warp takes (even).
template <typename T, int MODE, int kHeads>
__global__ void __launch_bounds__(kNrThreads) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  const int lane = threadIdx.x & 31, l = lane & 15, hi = lane >> 4;
  const int per = p.chunks[0] + p.chunks[1];
  const int64_t item = (int64_t)blockIdx.x * (kNrThreads / 32) + (threadIdx.x >> 5);
  griddep_wait();
  griddep_launch_dependents();
  if (item >= (int64_t)p.B * p.T * per) return;
  const int64_t tok = item / per;
  const int c = (int)(item - tok * per);
  const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
  const int side = c >= p.chunks[0];
  const int h0 = (side ? c - p.chunks[0] : c) * kHeads;
  const int64_t pi = (int64_t)b * p.ps_b + (int64_t)t * p.ps_t;
  const int64_t pos = !p.pos ? 0 : p.pos64 ? static_cast<const int64_t*>(p.pos)[pi] : (int64_t) static_cast<const int32_t*>(p.pos)[pi];
  const T* x = static_cast<const T*>(p.x[side]) + b * p.xs[side][0] + t * p.xs[side][2] + 8 * l;
  T* y = static_cast<T*>(p.y[side]) + b * p.ys[side][0] + t * p.ys[side][2] + 8 * l;
  const bool vec = p.vec[side];
  uint4 raw[kHeads / 2];
#pragma unroll
  for (int i = 0; i < kHeads / 2; ++i) {
    const int h = h0 + 2 * i + hi;
    raw[i] = h < p.H[side] ? nr_load(x + h * p.xs[side][1], vec) : make_uint4(0, 0, 0, 0);
  }
  if (pos < 0) return;  // a padding row: not written
  if (pos >= p.max_pos) {
    if (lane == 0) hkv_flag_error(HKV_DEVERR_BAD_POSITION);
    return;
  }
  const int r = p.rot >> 1;
  const float* row = p.table + pos * p.table_stride;
  float w[8], cs[8], sn[8];  // adjacent: cs/sn[0..3] serve the lane's four pairs
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = 1.f;
  if (p.w[side]) {
    if (p.w_dtype[side] == DT<T>::id && (reinterpret_cast<uintptr_t>(p.w[side]) & 15) == 0) {
      nr_unpack<T>(__ldg(reinterpret_cast<const uint4*>(p.w[side]) + l), w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = load_any(p.w[side], p.w_dtype[side], 8 * l + e);
    }
  }
  if constexpr (MODE == kNrAdjacent) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * l + e;
      cs[e] = i < r ? __ldg(row + i) : 1.f;
      sn[e] = i < r ? __ldg(row + r + i) : 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * l + e, i = d < r ? d : d - r;
      cs[e] = d < 2 * r ? __ldg(row + i) : 1.f;
      sn[e] = d < r ? -__ldg(row + r + i) : d < 2 * r ? __ldg(row + r + i) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads / 2; ++i) {
    const int h = h0 + 2 * i + hi;
    float v[8];
    nr_unpack<T>(raw[i], v);
    float rn = 1.f;
    if (p.w[side]) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(v[e], v[e], s);
#pragma unroll
      for (int k = 1; k < 16; k <<= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
      rn = rsqrtf(s * (1.f / HKV_D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= rn * w[e];
    }
    float o[8];
    if constexpr (MODE == kNrAdjacent) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool turned = 4 * l + e < r;  // the rest passes through, infinities included
        o[2 * e] = turned ? v[2 * e] * cs[e] - v[2 * e + 1] * sn[e] : v[2 * e];
        o[2 * e + 1] = turned ? v[2 * e + 1] * cs[e] + v[2 * e] * sn[e] : v[2 * e + 1];
      }
    } else if constexpr (MODE == kNrLane) {
      const int k = r >> 3;  // lanes between the halves of a pair
      const int from = l < k ? l + k : l < 2 * k ? l - k : l;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_sync(0xffffffffu, v[e], (lane & 16) | from);
        o[e] = l < 2 * k ? v[e] * cs[e] + other * sn[e] : v[e];
      }
    } else {
      const T* xr = x - 8 * l + (int64_t)h * p.xs[side][1];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * l + e, q = d < r ? d + r : d < 2 * r ? d - r : d;
        float other = 0.f;
        if (h < p.H[side] && d < 2 * r) {
          other = to_f32(xr[q]);
          if (p.w[side]) other *= rn * load_any(p.w[side], p.w_dtype[side], q);
        }
        o[e] = d < 2 * r ? v[e] * cs[e] + other * sn[e] : v[e];
      }
      __syncwarp();  // in place: the row's values are all read before the first is written
    }
    if (h >= p.H[side]) continue;
    T* yr = y + h * p.ys[side][1];
    if (vec) {
      *reinterpret_cast<uint4*>(yr) = make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]), pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) yr[e] = from_f32<T>(o[e]);
    }
  }
}

}  // namespace hkv
