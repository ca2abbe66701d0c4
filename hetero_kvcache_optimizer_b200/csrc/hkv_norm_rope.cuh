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
// warp's rows are in flight before the first is used. With rot = 128 a lane holds
// both halves of four pairs instead (two 8-byte loads: no exchange, one unpacking,
// 145 -> 124 us below); with another rot % 16 == 0 a pair's other half is 8 k dims
// away and sits in the same register of another lane (one shuffle); other sizes read
// it from the row again (L1).
// Measured: 32,768 tokens of 32 + 8 heads 124 us = 5.5 TB/s (a kernel that only copies
// the same rows: 107 us), 4,096 tokens of 28 + 4 heads 16.7 us, 8 tokens of 32 + 8
// heads 2.4 us (a launch). 61 warp instructions a row keep 60 % of the issue slots busy (76
// with 28 + 4 heads, which leave 8 of 40 places empty). The other rotations of the 32,768
// tokens: 64 of 128 dims by halves 150 us, 96 of 128 155, neighbours 137 (64) and 139 (128);
// 50 of 128 by halves, read twice, 446.
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
  int table_vec;           // table rows and their halves 16-byte aligned
  float eps;
  int B, T;
  uint32_t items;          // warps' pieces of work
  int chunks[2];           // warps per token of q and of k
};

constexpr int kNrThreads = 256;

// Half-split pairs whose halves are whole lanes apart | pairs of neighbours | any other half-split
// | half-split pairs over the whole head (rot = 128): a lane holds both halves of four pairs
enum { kNrLane = 0, kNrAdjacent = 1, kNrAny = 2, kNrWhole = 3 };

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

// Four values from `p` and four from `p + 64`.
template <typename T>
__device__ __forceinline__ uint4 nr_load2(const T* p, bool vec) {
  uint2 a, b;
  if (vec) {
    a = *reinterpret_cast<const uint2*>(p);
    b = *reinterpret_cast<const uint2*>(p + 64);
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    a = make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
    b = make_uint2((uint32_t)h[64] | ((uint32_t)h[65] << 16), (uint32_t)h[66] | ((uint32_t)h[67] << 16));
  }
  return make_uint4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ void nr_ld4(const float* p, float* v) {
  const float4 x = __ldg(reinterpret_cast<const float4*>(p));
  v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}

// One warp: heads h0 .. h1 - 1 (at most kHeads) of side SIDE (0 q, 1 k) of token (b, t). With rn the row's factor, out = rn (x (w c) + x' (w' s)), x' and w' the
// pair's other half: the products with the weights are made once for all heads, and
// x' is exchanged as it was loaded (16 bits), beside the sum of squares.
template <typename T, int MODE, int kHeads, int SIDE>
__device__ __forceinline__ void nr_rows(const NormRopeParams& p, int b, int t, int h0, int h1, int lane) {
  const int l = lane & 15, hi = lane >> 4;
  const int64_t pi = (int64_t)b * p.ps_b + (int64_t)t * p.ps_t;
  const int64_t pos = !p.pos ? 0 : p.pos64 ? static_cast<const int64_t*>(p.pos)[pi] : (int64_t) static_cast<const int32_t*>(p.pos)[pi];
  constexpr bool kWhole = MODE == kNrWhole;
  constexpr int kPer = kWhole ? 4 : 8;  // neighbouring values of a lane
  const T* x = static_cast<const T*>(p.x[SIDE]) + b * p.xs[SIDE][0] + t * p.xs[SIDE][2] + (int64_t)(h0 + hi) * p.xs[SIDE][1] + kPer * l;
  const int64_t xstep = 2 * p.xs[SIDE][1];
  const bool vec = p.vec[SIDE];
  uint4 raw[kHeads / 2];
  const T* xn = x;
#pragma unroll
  for (int i = 0; i < kHeads / 2; ++i, xn += xstep)
    raw[i] = h0 + 2 * i + hi < h1 ? (kWhole ? nr_load2(xn, vec) : nr_load(xn, vec)) : make_uint4(0, 0, 0, 0);
  if (pos < 0) return;  // a padding row: not written
  if (pos >= p.max_pos) {
    if (lane == 0) hkv_flag_error(HKV_DEVERR_BAD_POSITION);
    return;
  }
  const int r = p.rot >> 1;
  const float* row = p.table + pos * p.table_stride;
  const void* wp = p.w[SIDE];
  float w[8], cs[8], sn[8];  // adjacent: cs/sn[0 .. 3] serve the lane's four pairs
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = cs[e] = 1.f, sn[e] = 0.f;
  if (wp) {
    if (p.w_dtype[SIDE] == DT<T>::id && (reinterpret_cast<uintptr_t>(wp) & 15) == 0) {
      if constexpr (kWhole) {
        const uint2 a = __ldg(reinterpret_cast<const uint2*>(wp) + l), c = __ldg(reinterpret_cast<const uint2*>(wp) + 16 + l);
        nr_unpack<T>(make_uint4(a.x, a.y, c.x, c.y), w);
      } else {
        nr_unpack<T>(__ldg(reinterpret_cast<const uint4*>(wp) + l), w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = load_any(wp, p.w_dtype[SIDE], kWhole ? 4 * l + (e & 3) + 16 * (e & 4) : 8 * l + e);
    }
  }
  const int k = r >> 3;  // kNrLane: lanes between the halves of a pair
  const int from = (lane & 16) | (l < k ? l + k : l < 2 * k ? l - k : l);
  const bool turned = MODE == kNrAdjacent ? 4 * l < r : 8 * l < 2 * r;  // some of the lane's values
  if constexpr (kWhole) {
    if (p.table_vec) {
      nr_ld4(row + 4 * l, cs);
      nr_ld4(row + 64 + 4 * l, sn);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) cs[e] = __ldg(row + 4 * l + e), sn[e] = __ldg(row + 64 + 4 * l + e);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cs[e + 4] = cs[e] * w[e + 4];
      sn[e + 4] = sn[e] * w[e];
      cs[e] *= w[e];
      sn[e] *= -w[e + 4];
    }
  } else if constexpr (MODE == kNrAdjacent) {
    if (p.table_vec) {  // r is a multiple of 4: the lane's four pairs turn together or not at all
      if (turned) {
        nr_ld4(row + 4 * l, cs);
        nr_ld4(row + r + 4 * l, sn);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * l + e < r) cs[e] = __ldg(row + 4 * l + e), sn[e] = __ldg(row + r + 4 * l + e);
    }
  } else if (MODE == kNrLane && p.table_vec) {  // r is a multiple of 8: a lane's values are in one half
    if (turned) {
      const float* c = row + (8 * l < r ? 8 * l : 8 * l - r);
      nr_ld4(c, cs);
      nr_ld4(c + 4, cs + 4);
      nr_ld4(c + r, sn);
      nr_ld4(c + r + 4, sn + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) sn[e] = 8 * l < r ? -sn[e] : sn[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * l + e, i = d < r ? d : d - r;
      if (d < 2 * r) cs[e] = __ldg(row + i), sn[e] = d < r ? -__ldg(row + r + i) : __ldg(row + r + i);
    }
  }
  // the weights into the rotation
  if constexpr (MODE == kNrLane) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sn[e] *= __shfl_sync(0xffffffffu, w[e], from);
      cs[e] *= w[e];
    }
  } else if constexpr (MODE == kNrAny) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * l + e;
      if (wp && d < 2 * r) sn[e] *= load_any(wp, p.w_dtype[SIDE], d < r ? d + r : d - r);
      cs[e] *= w[e];
    }
  }
  T* yi = static_cast<T*>(p.y[SIDE]) + b * p.ys[SIDE][0] + t * p.ys[SIDE][2] + (int64_t)(h0 + hi) * p.ys[SIDE][1] + kPer * l;
  const int64_t ystep = 2 * p.ys[SIDE][1];
  const T* xi = x - 8 * l;
#pragma unroll
  for (int i = 0; i < kHeads / 2; ++i, yi += ystep, xi += xstep) {
    const bool on = h0 + 2 * i + hi < h1;
    float v[8], o[8];
    nr_unpack<T>(raw[i], v);
    float rn = 1.f;
    if (wp) {
      float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 8; e += 2) s2 = __ffma2_rn(make_float2(v[e], v[e + 1]), make_float2(v[e], v[e + 1]), s2);
      float s = s2.x + s2.y;
#pragma unroll
      for (int q = 1; q < 16; q <<= 1) s += __shfl_xor_sync(0xffffffffu, s, q);
      rn = rsqrtf(s * (1.f / HKV_D) + p.eps);
    }
    if constexpr (kWhole) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 z = __fmul2_rn(make_float2(v[e ^ 4], v[(e + 1) ^ 4]), make_float2(sn[e], sn[e + 1]));
        const float2 u = __ffma2_rn(make_float2(v[e], v[e + 1]), make_float2(cs[e], cs[e + 1]), z);
        o[e] = u.x, o[e + 1] = u.y;
      }
    } else if constexpr (MODE == kNrAdjacent) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = v[2 * e] * w[2 * e], c = v[2 * e + 1] * w[2 * e + 1];
        const bool on_pair = 4 * l + e < r;  // the rest passes through, infinities included
        o[2 * e] = on_pair ? a * cs[e] - c * sn[e] : a;
        o[2 * e + 1] = on_pair ? c * cs[e] + a * sn[e] : c;
      }
    } else if constexpr (MODE == kNrLane) {
      uint4 po;  // the pairs' other halves; nothing (not an infinity) where a lane passes through
      po.x = __shfl_sync(0xffffffffu, raw[i].x, from);
      po.y = __shfl_sync(0xffffffffu, raw[i].y, from);
      po.z = __shfl_sync(0xffffffffu, raw[i].z, from);
      po.w = __shfl_sync(0xffffffffu, raw[i].w, from);
      if (!turned) po = make_uint4(0, 0, 0, 0);
      nr_unpack<T>(po, o);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 z = __fmul2_rn(make_float2(o[e], o[e + 1]), make_float2(sn[e], sn[e + 1]));
        const float2 u = __ffma2_rn(make_float2(v[e], v[e + 1]), make_float2(cs[e], cs[e + 1]), z);
        o[e] = u.x, o[e + 1] = u.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * l + e;
        o[e] = v[e] * cs[e];
        if (on && d < 2 * r) o[e] = fmaf(to_f32(xi[d < r ? d + r : d - r]), sn[e], o[e]);
      }
      __syncwarp();  // in place: the row's values are all read before the first is written
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 u = __fmul2_rn(make_float2(o[e], o[e + 1]), make_float2(rn, rn));
      o[e] = u.x, o[e + 1] = u.y;
    }
    if (!on) continue;
    if constexpr (kWhole) {
      if (vec) {
        *reinterpret_cast<uint2*>(yi) = make_uint2(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]));
        *reinterpret_cast<uint2*>(yi + 64) = make_uint2(pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) yi[(e & 3) + 16 * (e & 4)] = from_f32<T>(o[e]);
      }
    } else if (vec) {
      *reinterpret_cast<uint4*>(yi) = make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]), pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) yi[e] = from_f32<T>(o[e]);
    }
  }
}

// Five CTAs an SM for whole heads, although 48 registers spill a little with eight heads a
// warp (96 bytes of stores, 24 of loads a thread): 16.7 against 18.1 us for a chunk with four
// CTAs, 124 against 133 for a prompt.
template <typename T, int MODE, int kHeads>
__global__ void __launch_bounds__(kNrThreads, MODE == kNrAny ? 2 : MODE == kNrWhole ? 5 : 4) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  const uint32_t item = blockIdx.x * (kNrThreads / 32) + (threadIdx.x >> 5);
  griddep_wait();
  griddep_launch_dependents();
  if (item >= p.items) return;
  const uint32_t per = p.chunks[0] + p.chunks[1], tok = item / per;
  const int c = (int)(item - tok * per), b = (int)(tok / (uint32_t)p.T), t = (int)(tok - (uint32_t)b * p.T), lane = threadIdx.x & 31;
  const int h0 = (c < p.chunks[0] ? c : c - p.chunks[0]) * kHeads;
  if (c < p.chunks[0]) nr_rows<T, MODE, kHeads, 0>(p, b, t, h0, min(p.H[0], h0 + kHeads), lane);
  else nr_rows<T, MODE, kHeads, 1>(p, b, t, h0, min(p.H[1], h0 + kHeads), lane);
}

}  // namespace hkv
