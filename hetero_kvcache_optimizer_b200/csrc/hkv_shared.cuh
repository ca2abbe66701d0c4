// Decode attention over an INT4 prefix that several sequences share.
// Included by hetero_kv.cu.
//
// A group of n sequences has one prefix; per KV head its n G query heads are the
// columns of ONE product over the prefix's tokens, so the packed pages are read
// and dequantised once per row tile of N = 32, 64 or 128 rows instead of once per
// sequence (at most 16 rows, and outputs finer than bf16: shared_rows_kernel below):
//   S^T[token][row] = K Q^T,  P = 2^(S qscale - m),  O^T[dim][row] += V^T P
// on tcgen05 with the tokens (then the dims) as the MMA's M = 128 and the rows as
// its N: a decode batch has few rows, and this way they cost what they are (with
// the rows as M, 32 of them would cost 128, and the exponentials would sit in one
// warp). The running max m and the sum of P are fp32; m moves only when a score
// beats it by more than 2^8. K, V and P are rounded to f16, the type of their MMA:
// K and V where they are dequantised (2^-11 relative; ref's f32 scale enters K as the
// sum of two f16 and V rounded), P in (0, 2^8]; with key channels ten times as large
// as the rest that leaves the output 4e-4 to 1.4e-3 off in the 2-norm,
// below the 1.7e-3 of a bf16 output's own rounding; other outputs do not come here.
//
// A grid of p.C persistent CTAs; every (group, KV head, row tile) unit's 128-token
// tiles, with a charge of kShCharge tiles per unit for a piece's start and end,
// are cut into equal ranges, one per CTA (so a CTA has a few "pieces", runs of
// tiles of one unit). Each piece leaves un-normalised partials (O, m, l) at index
// cta + unit (unique: each next piece raises one of the two), and
// shared_merge_kernel joins a row's partials with the one of its own tokens.
//
// Roles (tile n of the CTA uses the buffers n mod their number):
//   softmax   thread = token, 32 of the tile's rows, 16 at a time: S^T from TMEM, P as f16
//             rows [token][row] (N-major B of O^T)
//   K warps   thread = token: dequantised f16 K straight into TMEM (A of S^T, so
//             K does not cross shared memory again)
//   V warps   dequantised V^T into shared memory (128-byte swizzle, A of O^T)
//   producer  one bulk copy per packed 128-token block into a ring of raw slots
//   two MMA warps  one issues S^T, up to two tiles ahead, the other O^T: one thread
//             for both held S^T(n + 2) back until P(n) was written
// Every wait is bounded (HKV_WAIT_NS); on expiry the device error word is set, the
// CTA's roles leave, and copies and products in flight are waited for before TMEM
// is freed.
//
// Measured (65,536 tokens, 8 KV heads, fp16min g32, all SMs, prefix and merge alone):
// 32 rows 44.3 us, 64 rows 55.3, 128 rows 74.1, 256 rows 127.8 (538 TFLOP/s), of which
// about 10 us are start and end. The steady state is 1.25 / 1.65 / 2.3 us per tile and
// SM, bound by none of its resources alone: at 32 rows 5,190 warp instructions a tile
// (the whole launch's over its tiles; about 2,180 unpack K and V), 56 % of the issue
// slots, 11 % of the tensor pipe and 16 % of shared memory's wavefronts busy (ref, group
// 32: 7,000 instructions, 54, 8 and 25 %); at 128 rows 8,180, 61, 30 and 32 %. Steps that counted: K through TMEM, one
// elected thread for the MMAs (57 -> 10 cycles to issue one), one polling warp a role,
// half-size V code.
#pragma once
#include "hkv_prefill.cuh"

namespace hkv {

constexpr int kShMaxGroups = 512;
constexpr int kShCharge = 6;
constexpr int kShRawBytes = 21504;  // the largest block (ref, group 32)

// Up to 64 rows, even and odd tiles of a CTA are two streams, each with its own
// softmax warps, running max, O and partial: two tiles' softmax are in flight at a
// time, neither waiting for the other's rescale. At 128 rows TMEM has room for one.
constexpr int sh_streams(int n) { return n <= 64 ? 2 : 1; }
constexpr int sh_col_groups(int n) { return n <= 32 ? 1 : n <= 64 ? 2 : 4; }  // softmax groups that share a tile's rows
constexpr int sh_softmax_groups(int n) { return sh_streams(n) * sh_col_groups(n); }
// Sets of four V warps, a tile each in turn (65,536 tokens, 8 heads: 44.2 us for 32 rows, one set
// 47.0; 55.6 us for 64 rows, two sets 58.3: their registers are missed by the softmax).
constexpr int sh_v_sets(int n) { return n <= 32 ? 2 : 1; }
constexpr int sh_threads(int n) { return 32 * (4 * (sh_softmax_groups(n) + 1 + sh_v_sets(n)) + 3); }
constexpr int sh_slots(int n) { return n <= 32 ? 4 : n <= 64 ? 3 : 2; }
constexpr int sh_v_bufs(int n) { return n <= 64 ? 3 : 2; }
constexpr int sh_p_row(int n) { return n <= 32 ? 64 : 128; }  // bytes of a token's row of P, swizzled as wide
constexpr int sh_p_bytes(int n) { return 128 * sh_p_row(n) * (n <= 64 ? 1 : 2); }  // [row block of 64][token]
constexpr int sh_smem(int n) {  // Q | Vt | P[2] | raw slots | alignment
  return n * 256 + sh_v_bufs(n) * kPfTileBytes + 2 * sh_p_bytes(n) + sh_slots(n) * kShRawBytes + 1024;
}
constexpr int sh_tmem_cols(int n) { return 128 + (2 + sh_streams(n)) * n <= 256 ? 256 : 512; }  // K[2] | S[2] | O[streams]

struct SharedParams {
  const void* q;
  int q_dtype;
  int64_t q_sb, q_sh;
  int q_pairs;              // pairs of query values are 4-byte aligned
  hkv_int4_store prefix;    // batch = groups
  int P, Hkv, G, C;         // groups, KV heads, query heads per KV head, CTAs
  float qscale;             // sm_scale * log2(e)
  float* part_o;            // [C + units][ns][N][128]
  float* part_ml;           // [C + units][ns][N][2]
  // merge
  const float* own_o;       // [B][Hq][128], or NULL
  const float* own_ml;      // [B][Hq][2]
  void* out;
  int out_dtype;
  int64_t out_sb, out_sh;
  int B, N, ns;             // N: rows of a row tile; ns: partials of a piece
  int start[kShMaxGroups + 1];  // sequences [start[p], start[p + 1]) are group p
};

// The schedule of a launch, from the device lengths: steps before group p.
__device__ __forceinline__ int sh_len(const SharedParams& p, int g) {
  return min(p.prefix.max_pages * p.prefix.page_tokens, max(0, p.prefix.lengths ? p.prefix.lengths[g] : p.prefix.len));
}
__device__ __forceinline__ int sh_row_tiles(const SharedParams& p, int g) {
  return ((p.start[g + 1] - p.start[g]) * p.G + p.N - 1) / p.N;
}
__device__ __forceinline__ int sh_units(const SharedParams& p, int g) { return p.Hkv * sh_row_tiles(p, g); }

struct ShGroup {
  int step, unit;  // steps and units before the group
  int len;         // its prefix's length
};
// Fills s_g[0 .. P] (one warp); s_g[P].step is the launch's step count.
__device__ __forceinline__ void sh_schedule(const SharedParams& p, ShGroup* s_g) {
  const int lane = threadIdx.x & 31;
  int step = 0, unit = 0;
  for (int g0 = 0; g0 <= p.P; g0 += 32) {
    const int g = g0 + lane;
    int st = 0, un = 0, len = 0;
    if (g < p.P) {
      len = sh_len(p, g);
      const int tiles = (len + HKV_BLOCK_TOKENS - 1) / HKV_BLOCK_TOKENS;
      un = sh_units(p, g);
      st = tiles > 0 ? un * (tiles + kShCharge) : 0;
    }
    int si = st, ui = un;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, si, k), b = __shfl_up_sync(0xffffffffu, ui, k);
      if (lane >= k) si += a, ui += b;
    }
    if (g <= p.P) s_g[g] = ShGroup{step + si - st, unit + ui - un, len};
    step += __shfl_sync(0xffffffffu, si, 31);
    unit += __shfl_sync(0xffffffffu, ui, 31);
  }
}
// First step of CTA c's range.
__device__ __forceinline__ int sh_cut(int total, int C, int c) { return (int)((int64_t)total * c / C); }

struct ShPiece {
  int g, h, rt;  // group, KV head, row tile
  int unit;      // ordinal of the unit
  int t0, n;     // tiles [t0, t0 + n)
};
// A unit's tile i is step base + kShCharge + i; the first piece of the steps
// [at, end) (n == 0: none), `at` moved behind its unit.
__device__ __forceinline__ ShPiece sh_next(const SharedParams& p, const ShGroup* s_g, int& at, int end) {
  ShPiece r;
  r.n = 0;
  int g = 0;
  while (at < end) {
    while (g < p.P && s_g[g + 1].step <= at) ++g;
    if (g >= p.P) break;
    const int units = s_g[g + 1].unit - s_g[g].unit;
    const int per = (s_g[g + 1].step - s_g[g].step) / units;
    const int u = (at - s_g[g].step) / per, base = s_g[g].step + u * per + kShCharge;
    const int lo = max(at - base, 0), hi = min(per - kShCharge, end - base);
    at = base + per - kShCharge;
    if (hi > lo) {
      const int rts = units / p.Hkv;
      r.g = g;
      r.h = u / rts;
      r.rt = u - r.h * rts;
      r.unit = s_g[g].unit + u;
      r.t0 = lo;
      r.n = hi - lo;
      break;
    }
  }
  return r;
}

// N-major B descriptor: a token's row of 64 f16 (128 bytes, 128-byte swizzle; the
// second 64 columns 16 KiB further) or of 32 (64 bytes, 64-byte swizzle), 8 rows a group.
__device__ __forceinline__ uint64_t sh_desc_n(uint32_t addr, int row) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(row * 8 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)(row == 64 ? 4 : 2) << 61);
}
constexpr uint32_t sh_idesc(int n, bool b_n_major) {
  return (1u << 4) | (b_n_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void sh_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void sh_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void sh_ld(uint32_t addr, float (&v)[16]) {  // 16 columns of this thread's lane
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void sh_st(uint32_t addr, const float (&v)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
  tm_st16u(addr, r);
}
__device__ __forceinline__ bool bar_or(int id, int n, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, %2, %3, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}

// One lane of a converged warp, in a form by which the compiler knows that a
// single thread follows: under `lane == 0` each tcgen05.mma was issued through a
// loop over the active lanes, 57 cycles apiece instead of 10.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}

// Bounded wait for a phase. The loop is out of line: with a copy at each of fifteen
// places the roles' code missed the instruction cache (64 rows: 64.6 -> 56.5 us).
__device__ __noinline__ bool sh_wait_long(uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity); }
__device__ __forceinline__ bool sh_wait(uint64_t* bar, uint32_t parity) {
  return mbar_try_wait(bar, parity & 1u) || sh_wait_long(bar, parity & 1u);
}

// Query values i and i + 1 as two f16 (bf16 rounded to them).
__device__ __forceinline__ uint32_t sh_q2(const SharedParams& p, int64_t i) {
  if (!p.q_pairs) return h2u(__floats2half2_rn(load_any(p.q, p.q_dtype, i), load_any(p.q, p.q_dtype, i + 1)));
  const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + i);
  return p.q_dtype == HKV_DT_F16 ? w : h2u(__float22half2_rn(__bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w))));
}

// Dims of 16-byte chunk kc (8 values) of Q's and K's common order: value 2 c + e
// is dim 32 (kc / 4) + 8 c + 2 (kc % 4) + e, the order in which nib8_to_h2 yields
// a K token's words, so that K needs no shuffling on its way into TMEM.
__device__ __forceinline__ int sh_dim(int kc, int c) { return 32 * (kc >> 2) + 8 * c + 2 * (kc & 3); }

// K of token t (thread t) of the raw block into TMEM lane t, columns 0 .. 63. The
// token's four 16-byte chunks are read in an order rotated by t / 2, so that the 8
// threads of a load phase hit 8 distinct bank groups, and rotated back with selects.
template <int FMT, int GROUP>
__device__ __forceinline__ void sh_convert_k(const uint8_t* rb, uint32_t tmem, int t, bool valid) {
  constexpr int NG = HKV_D / GROUP;
  const int rot = (t >> 1) & 3;
  const bool r1 = rot & 1, r2 = rot & 2;
  const uint8_t* meta = rb + HKV_META_OFF;
  uint32_t v[4][4], u[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 c = *reinterpret_cast<const uint4*>(rb + t * 64 + (((j + rot) & 3) << 4));
    v[j][0] = c.x, v[j][1] = c.y, v[j][2] = c.z, v[j][3] = c.w;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int w = 0; w < 4; ++w) u[j][w] = r1 ? v[(j + 3) & 3][w] : v[j][w];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int w = 0; w < 4; ++w) v[j][w] = r2 ? u[(j + 2) & 3][w] : u[j][w];
  __half ks[NG], km[NG];
  if constexpr (FMT == HKV_FMT_FP16MIN) vload_h<NG>(meta + 2 * NG * t, ks), vload_h<NG>(meta + 256 * NG + 2 * NG * t, km);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t o[32];
#pragma unroll
    for (int w2 = 0; w2 < 2; ++w2) {  // dims 32 w .. + 31
      const int w = 2 * half + w2, g = w * 32 / GROUP;
      __half2 s2, m2;  // ref: the f32 scale as the sum of two f16
      uint32_t zlo = 0, zhi = 0;
      if constexpr (FMT == HKV_FMT_FP16MIN) {
        s2 = __half2half2(ks[g]);
        m2 = __half2half2(km[g]);
      } else {
        const uint32_t z = meta[1024 * NG + t * NG + g];
        const float s = reinterpret_cast<const float*>(meta)[t * NG + g];
        s2 = __float2half2_rn(s);
        m2 = __float2half2_rn(s - __low2float(s2));
        zlo = h2u(__float2half2_rn(1024.f + (float)z));
        zhi = h2u(__float2half2_rn(-64.f - (float)z));
      }
      if (!valid) s2 = m2 = __float2half2_rn(0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h[4];
        if constexpr (FMT == HKV_FMT_FP16MIN) nib8_to_h2(v[j][w], h);
        else nib8_to_h2_z(v[j][w], zlo, zhi, h);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          o[16 * w2 + 4 * j + c] = h2u(__hfma2(u2h(h[c]), s2, FMT == HKV_FMT_FP16MIN ? m2 : __hmul2(u2h(h[c]), m2)));
      }
    }
    tm_st32u(tmem + 32 * half, o);
  }
  tm_wait_st();
}

// V of the raw block into sVt ([dim][token], 128-byte swizzle): thread (o, k2, i) has
// tokens 8 o .. 8 o + 7 (and 64 on) and words 2 k2, 2 k2 + 1 of chunk i of their four
// pairs, so the 16 threads of a load phase read a pair's 128 bytes and the 8 of a
// store phase hit 8 chunks apart. Word k of chunk i holds dims i + 32 k + 8 m (nibble m) of a pair's two tokens. Tokens at and behind
// `valid` become zero (their P is zero and their bytes may be any bits).
template <int FMT, int GROUP>
__device__ __forceinline__ void sh_convert_v(const uint8_t* rb, uint8_t* sVt, int t, int valid) {
  constexpr int NG = HKV_D / GROUP;
  const int i = t & 7, o0 = t >> 4, k2 = (t >> 3) & 1;
  const uint8_t* meta = rb + HKV_META_OFF;
#pragma unroll 1  // half the code: the roles share the instruction cache
  for (int rep = 0; rep < 2; ++rep) {
    const int o = o0 + 8 * rep;
    uint2 cw[4];
    __half2 vs2[4][2], vm2[4][2];  // fp16min: scales and mins of the pairs in the groups of words 2 k2, 2 k2 + 1
#pragma unroll
    for (int pp = 0; pp < 4; ++pp) {
      cw[pp] = *reinterpret_cast<const uint2*>(rb + HKV_V_CODES_OFF + v_chunk_off(4 * o + pp, i) + 8 * k2);
      if constexpr (FMT == HKV_FMT_FP16MIN) {
        const uint8_t* mp = meta + 512 * NG + 4 * ((4 * o + pp) * NG + 64 * k2 / GROUP);
        if constexpr (NG == 4) {
          vload_h2<2>(mp, vs2[pp]);
          vload_h2<2>(mp + 256 * NG, vm2[pp]);
        } else {
          vs2[pp][0] = vs2[pp][1] = *reinterpret_cast<const __half2*>(mp);
          vm2[pp][0] = vm2[pp][1] = *reinterpret_cast<const __half2*>(mp + 256 * NG);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int k = 2 * k2 + w, g = 32 * k / GROUP;
      uint32_t h[4][4];  // [pair][nibble m], then the values
#pragma unroll
      for (int pp = 0; pp < 4; ++pp) {
        const int q = 4 * o + pp;  // tokens 2 q, 2 q + 1
        __half2 s2, m2;
        const uint32_t wd = w ? cw[pp].y : cw[pp].x;
        if constexpr (FMT == HKV_FMT_FP16MIN) {
          s2 = vs2[pp][w];
          m2 = vm2[pp][w];
        } else {
          const float* vs = reinterpret_cast<const float*>(meta + 512 * NG);
          s2 = __floats2half2_rn(vs[2 * q * NG + g], vs[(2 * q + 1) * NG + g]);
          m2 = __float2half2_rn(0.f);
        }
        if (valid < HKV_BLOCK_TOKENS) {
          const uint32_t keep = (2 * q < valid ? 0x0000FFFFu : 0u) | (2 * q + 1 < valid ? 0xFFFF0000u : 0u);
          s2 = u2h(h2u(s2) & keep);
          m2 = u2h(h2u(m2) & keep);
        }
        if constexpr (FMT == HKV_FMT_FP16MIN) {
          nib8_to_h2(wd, h[pp]);
        } else {
          const uint8_t* vz = meta + 1152 * NG;
          const float za = (float)vz[2 * q * NG + g], zb = (float)vz[(2 * q + 1) * NG + g];
          nib8_to_h2_z(wd, h2u(__floats2half2_rn(1024.f + za, 1024.f + zb)), h2u(__floats2half2_rn(-64.f - za, -64.f - zb)), h[pp]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) h[pp][m] = h2u(__hfma2(u2h(h[pp][m]), s2, m2));
      }
#pragma unroll
      for (int m = 0; m < 4; ++m)  // dim i + 32 k + 8 m: its row is 0 mod 8 plus i
        *reinterpret_cast<uint4*>(sVt + pf_chunk(i, o) + (32 * k + 8 * m) * 128) = make_uint4(h[0][m], h[1][m], h[2][m], h[3][m]);
    }
  }
}

template <int FMT, int GROUP, int N>
__global__ void __launch_bounds__(sh_threads(N), 1) shared_prefix_kernel(const __grid_constant__ SharedParams p) {
  constexpr int NS = sh_streams(N), CG = sh_col_groups(N);
  constexpr int SG = NS * CG;                // softmax groups of 128 threads
  constexpr int COLS = N / CG;               // columns of a softmax thread
  constexpr int SUB = 16;  // taken at a time
  constexpr int VB = sh_v_bufs(N), PR = sh_p_row(N);
  constexpr int VS = sh_v_sets(N);
  constexpr int R = sh_slots(N);
  constexpr int kThreads = sh_threads(N);
  constexpr uint32_t kBlock = block_bytes(FMT, GROUP);
  constexpr uint32_t kCols = sh_tmem_cols(N);
  extern __shared__ __align__(1024) uint8_t sh_raw[];
  __shared__ __align__(8) uint64_t raw_full[R], raw_free[R], k_full[2], v_full[VB], v_free[VB], s_full[2], s_free[2];
  __shared__ __align__(8) uint64_t p_full[2], pv_done[2], q_full, drain[2];
  __shared__ uint32_t s_tmem;
  __shared__ ShGroup s_g[kShMaxGroups + 1];
  __shared__ int s_valid[16];        // tokens in use of tile n & 15
  __shared__ __align__(16) float s_ms[NS][N], s_fs[NS][N];  // column's running max; its last rescale
  __shared__ float s_cms[NS][4][N];  // per-warp column maxima, then sums
  uint8_t* sm = sh_raw + ((1024u - (smem_u32(sh_raw) & 1023u)) & 1023u);
  uint8_t* sQ = sm;
  uint8_t* sV = sQ + N * 256;
  uint8_t* sP = sV + VB * kPfTileBytes;
  uint8_t* raw = sP + 2 * sh_p_bytes(N);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;

  if (t == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_free[i], 8);
    }
    for (int i = 0; i < VB; ++i) {
      mbar_init(&v_full[i], 4);
      mbar_init(&v_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&s_free[i], 4 * CG);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4 * CG);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(&q_full, 4 * SG);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "n"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  griddep_launch_dependents();  // the own part may start beside this grid
  if (warp == 1) sh_schedule(p, s_g);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem, tS = tmem + 128, tO = tmem + 128 + 2 * N;
  const int total = s_g[p.P].step;
  int at = sh_cut(total, p.C, blockIdx.x);
  const int end = sh_cut(total, p.C, blockIdx.x + 1);
  uint32_t n0 = 0, pieces = 0;  // tiles and pieces of the CTA before this one
  uint32_t issued = 0;   // producer: copies; MMA warp: whether there are products
  bool ok = true;

  while (true) {
    const ShPiece pc = sh_next(p, s_g, at, end);
    if (pc.n == 0) break;
    const int rows = (p.start[pc.g + 1] - p.start[pc.g]) * p.G - pc.rt * N;
    if (warp < 4 * SG) {
      // ---------------- softmax: thread = token, columns [col0, col0 + COLS) of the stream's tiles ----------------
      const int sg = warp >> 2, tok = t & 127, col0 = sg % CG * COLS, stream = sg / CG;
      float *s_m = s_ms[stream], *s_f = s_fs[stream];
      auto s_cm = s_cms[stream];
      const uint32_t tOs = tO + stream * N;
      const int j0 = NS == 2 ? (n0 ^ stream) & 1 : 0;  // the stream's first tile
      // 16-byte chunk k of the thread's columns is at prow ^ 16 k (rows of 8 or 4 chunks, swizzled by the token)
      const uint32_t prow = smem_u32(sP) + (col0 >> 6) * 16384 + tok * PR +
                            (PR == 64 ? ((tok >> 1) & 3) << 4 : (((col0 & 63) >> 3) ^ (tok & 7)) << 4);
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const float2 qs2 = make_float2(p.qscale, p.qscale);
      // every group is through with the last piece's scores: its query rows make room
      // for this one's, in K's dim order (a group that gave up says so here)
      if (!bar_and(8, 128 * SG, ok)) break;
      for (int c = t; c < N * 16; c += 128 * SG) {
        const int n = c >> 4, kc = c & 15;
        uint32_t o[4] = {0u, 0u, 0u, 0u};
        if (n < rows) {
          const int r = pc.rt * N + n, sq = r / p.G;
          const int64_t base = (int64_t)(p.start[pc.g] + sq) * p.q_sb + (int64_t)(pc.h * p.G + r - sq * p.G) * p.q_sh;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = sh_q2(p, base + sh_dim(kc, e));
        }
        *reinterpret_cast<uint4*>(sQ + (kc >> 3) * (N * 128) + n * 128 + (((kc & 7) ^ (n & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      if (tok < COLS) s_m[col0 + tok] = -1.0e30f;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + sg) : "memory");
      float l[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) l[i] = 0.f;
      for (int j = j0; j < pc.n; j += NS) {
        const uint32_t n = n0 + j, buf = n & 1;
        // One warp of a role polls the mbarriers and the others sleep at a named
        // barrier: with every warp polling, two thirds of the instructions were polls.
        bool good = true;
        if ((warp & 3) == 0) {
          good = sh_wait(&s_full[buf], n >> 1);
          if (n >= 2) good = sh_wait(&pv_done[buf], (n >> 1) - 1) && good;  // P[buf] is free
          __syncwarp();
        }
        ok = bar_and(1 + sg, 128, good);
        if (!ok) break;
        tc_fence_after();
        const bool see = tok < s_valid[n & 15];
#pragma unroll
        for (int s0 = 0; s0 < COLS; s0 += SUB) {
          const int c0 = col0 + s0;
          const uint32_t ts = tS + buf * N + c0 + lanes;
          float x[SUB];  // S qscale - m
          auto scores = [&]() {
            sh_ld(ts, x);
#pragma unroll
            for (int i = 0; i < SUB; i += 4) {
              const float4 m = *reinterpret_cast<const float4*>(&s_m[c0 + i]);
              const float2 a = __ffma2_rn(make_float2(x[i], x[i + 1]), qs2, make_float2(-m.x, -m.y));
              const float2 b = __ffma2_rn(make_float2(x[i + 2], x[i + 3]), qs2, make_float2(-m.z, -m.w));
              x[i] = a.x, x[i + 1] = a.y, x[i + 2] = b.x, x[i + 3] = b.y;
            }
          };
          scores();
          float mx = fmaxf(x[0], x[SUB - 1]);
#pragma unroll
          for (int i = 1; i + 1 < SUB; i += 2) mx = fmax3(mx, x[i], x[i + 1]);
          if (bar_or(1 + sg, 128, see && mx > kPfLazy)) {  // a column's max moves
            sh_ld(ts, x);
            float mine = -INFINITY;  // the warp's max of column c0 + lane
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
              float v;
              asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(v) : "f"(see ? x[i] : -INFINITY));
              if (lane == i) mine = v;
            }
            if (lane < SUB) s_cm[warp & 3][c0 + lane] = mine * p.qscale;
            asm volatile("bar.sync %0, 128;" ::"r"(1 + sg) : "memory");
            if ((warp & 3) == 0 && lane < SUB) {
              const int c = c0 + lane;
              const float top = fmaxf(fmaxf(s_cm[0][c], s_cm[1][c]), fmaxf(s_cm[2][c], s_cm[3][c]));
              const float old = s_m[c], m = top > old + kPfLazy ? top : old;
              s_m[c] = m;
              s_f[c] = fast_exp2(old - m);
            }
            // the stream's last O has to be there before it is rescaled (with two streams
            // that is O(n - 2), waited for above)
            good = NS == 2 || (warp & 3) != 0 || j == 0 || sh_wait(&pv_done[buf ^ 1], (n - 1) >> 1);
            __syncwarp();
            ok = bar_and(1 + sg, 128, good);
            if (!ok) break;
            if (j > j0) {
              tc_fence_after();
              sh_ld(tOs + c0 + lanes, x);
#pragma unroll
              for (int i = 0; i < SUB; ++i) x[i] *= s_f[c0 + i];
              sh_st(tOs + c0 + lanes, x);
              tm_wait_st();
            }
#pragma unroll
            for (int i = 0; i < SUB; ++i) l[s0 + i] *= s_f[c0 + i];
            scores();
          }
          if (!see) {
#pragma unroll
            for (int i = 0; i < SUB; ++i) x[i] = -INFINITY;
          }
          if (s0 + SUB == COLS) {  // the last scores of the tile are read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[buf]);
          }
#pragma unroll
          for (int i = 0; i < SUB; i += 8) {
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float2 y = make_float2(fast_exp2(x[i + e]), fast_exp2(x[i + e + 1]));
              const float2 z = __fadd2_rn(make_float2(l[s0 + i + e], l[s0 + i + e + 1]), y);
              l[s0 + i + e] = z.x, l[s0 + i + e + 1] = z.y;
              pk[e >> 1] = h2u(__floats2half2_rn(y.x, y.y));
            }
            const uint32_t at16 = (prow + buf * sh_p_bytes(N)) ^ ((s0 + i) << 1);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at16), "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3]) : "memory");
          }
        }
        if (!ok) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      if (ok) {
        // the piece's partial: O^T from TMEM (lane = dim), m and l per column
        const int last = (int)(n0 + pc.n - 1) - (NS == 2 ? (int)((n0 + pc.n - 1) ^ stream) & 1 : 0);  // the stream's last tile
        const int64_t id = ((int64_t)(blockIdx.x + pc.unit) * NS + stream) * N;
        const bool any = last >= (int)n0, good = (warp & 3) != 0 || !any || sh_wait(&pv_done[last & 1], last >> 1);
        __syncwarp();
        ok = bar_and(1 + sg, 128, good);
        tc_fence_after();
        if (ok) {
#pragma unroll
          for (int s0 = 0; s0 < COLS; s0 += SUB) {
            float o[SUB];
            sh_ld(tOs + col0 + s0 + lanes, o);
#pragma unroll
            for (int i = 0; i < SUB; ++i)
              if (any && col0 + s0 + i < rows) p.part_o[(id + col0 + s0 + i) * HKV_D + tok] = o[i];
            // sums over the warp's tokens: lane ends with column lane % SUB
#pragma unroll
            for (int i = 0; i < SUB; ++i) o[i] = l[s0 + i] + __shfl_xor_sync(0xffffffffu, l[s0 + i], 16);
#pragma unroll
            for (int k = SUB / 2; k >= 1; k >>= 1) {
              const bool up = lane & k;
#pragma unroll
              for (int i = 0; i < k; ++i) {
                const float send = up ? o[i] : o[i + k], keep = up ? o[i + k] : o[i];
                o[i] = keep + __shfl_xor_sync(0xffffffffu, send, k);
              }
            }
            if (lane < SUB) s_cm[warp & 3][col0 + s0 + lane] = o[0];
          }
          asm volatile("bar.sync %0, 128;" ::"r"(1 + sg) : "memory");
          const int c = col0 + tok;
          if (tok < COLS && c < rows)
            *reinterpret_cast<float2*>(p.part_ml + (id + c) * 2) = make_float2(s_m[c], (s_cm[0][c] + s_cm[1][c]) + (s_cm[2][c] + s_cm[3][c]));
        }
      }
    } else if (warp < 4 * (SG + 1)) {
      // ---------------- K: thread = token = TMEM lane ----------------
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      for (int j = 0; j < pc.n; ++j) {
        const uint32_t n = n0 + j, buf = n & 1, slot = n % R;
        bool good = true;
        if ((warp & 3) == 0) {
          good = sh_wait(&raw_full[slot], n / R);
          if (n >= 2) good = sh_wait(&s_full[buf], (n >> 1) - 1) && good;  // S(n - 2) has read K[buf]
          __syncwarp();
        }
        ok = bar_and(5, 128, good);
        if (!ok) break;
        tc_fence_after();
        sh_convert_k<FMT, GROUP>(raw + slot * kShRawBytes, tmem + 64 * buf + lanes, t & 127, (t & 127) < s_valid[n & 15]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&k_full[buf]);
          mbar_arrive(&raw_free[slot]);
        }
      }
    } else if (warp < 4 * (SG + 1 + VS)) {
      // ---------------- V ----------------
      const int set = (warp - 4 * (SG + 1)) >> 2, vt = t & 127;
      for (int j = VS == 2 ? (n0 ^ set) & 1 : 0; j < pc.n; j += VS) {
        const uint32_t n = n0 + j, vb = n % VB, slot = n % R;
        bool good = true;
        if ((warp & 3) == 0) {
          good = sh_wait(&raw_full[slot], n / R);
          if (n >= VB) good = sh_wait(&v_free[vb], n / VB - 1) && good;  // O(n - VB) has read Vt[vb]
          __syncwarp();
        }
        ok = bar_and(6 + set, 128, good);
        if (!ok) break;
        sh_convert_v<FMT, GROUP>(raw + slot * kShRawBytes, sV + vb * kPfTileBytes, vt, s_valid[n & 15]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&v_full[vb]);
          mbar_arrive(&raw_free[slot]);
        }
      }
    } else if (warp == 4 * (SG + 1 + VS)) {
      // ---------------- producer ----------------
      const int u = pc.g * p.Hkv + pc.h;
      const int len = s_g[pc.g].len;
      int64_t ids = -1;
      for (int j = 0; j < pc.n; ++j) {
        const uint32_t n = n0 + j, slot = n % R;
        const int tok = (pc.t0 + j) * HKV_BLOCK_TOKENS;
        if ((j & 31) == 0) ids = j + lane < pc.n ? store_page(p.prefix, u, tok + lane * HKV_BLOCK_TOKENS) : -1;
        const int64_t page = __shfl_sync(0xffffffffu, ids, j & 31);
        if (n >= R && !__all_sync(0xffffffffu, sh_wait(&raw_free[slot], n / R - 1))) {
          ok = false;
          break;
        }
        if (lane == 0) {
          s_valid[n & 15] = page >= 0 ? min(HKV_BLOCK_TOKENS, len - tok) : 0;
          if (page >= 0) {
            const uint8_t* src = static_cast<const uint8_t*>(p.prefix.pages) + page * p.prefix.page_stride +
                                 (int64_t)((tok % p.prefix.page_tokens) / HKV_BLOCK_TOKENS) * kBlock;
            mbar_arrive_expect_tx(&raw_full[slot], kBlock);
            bulk_g2s(raw + slot * kShRawBytes, src, kBlock, &raw_full[slot]);
          } else {  // no such page: the tile counts as hidden, its bytes are the last tile's
            hkv_flag_error(HKV_DEVERR_BAD_PAGE);
            mbar_arrive(&raw_full[slot]);
          }
        }
        __syncwarp();
        issued = n + 1;
      }
      if (!ok)  // copies in flight land before the CTA ends
        for (uint32_t n = issued > R ? issued - R : 0; n < issued; ++n) sh_wait(&raw_full[n % R], n / R);
    } else if (warp == 4 * (SG + 1 + VS) + 1) {
      // ---------------- S^T(n) = K(n) Q^T, up to two tiles ahead of the softmax ----------------
      if (elect_one()) {
        const uint32_t q0 = smem_u32(sQ);
        ok = sh_wait(&q_full, pieces);
        for (int j = 0; ok && j < pc.n; ++j) {
          const uint32_t n = n0 + j, buf = n & 1;
          ok = sh_wait(&k_full[buf], n >> 1) && (n < 2 || sh_wait(&s_free[buf], (n >> 1) - 1));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            sh_mma_ts(tS + buf * N, tmem + 64 * buf + 8 * kk, pf_desc(q0 + (kk >> 2) * (N * 128) + (kk & 3) * 32),
                      sh_idesc(N, false), kk > 0);
          pf_commit(&s_full[buf]);
          issued = 1;
        }
        if (!ok && issued) {  // products in flight end before TMEM is freed
          pf_commit(&drain[0]);
          sh_wait(&drain[0], 0);
        }
      }
    } else if (elect_one()) {
      // ---------------- O^T += V^T P; a stream's O is overwritten once P of a piece's first
      // tile says that its groups have read the last piece's ----------------
      const uint32_t v0 = smem_u32(sV), p0 = smem_u32(sP);
      for (int j = 0; j < pc.n; ++j) {
        const uint32_t n = n0 + j, buf = n & 1, vb = n % VB;
        ok = sh_wait(&v_full[vb], n / VB) && sh_wait(&p_full[buf], n >> 1);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          sh_mma_ss(tO + (NS == 2 ? buf * N : 0), pf_desc(v0 + vb * kPfTileBytes + (kk >> 2) * 16384 + (kk & 3) * 32),
                    sh_desc_n(p0 + buf * sh_p_bytes(N) + kk * 16 * PR, PR), sh_idesc(N, true), j >= NS || kk > 0);
        pf_commit(&pv_done[buf]);
        pf_commit(&v_free[vb]);
        issued = 1;
      }
      if (!ok && issued) {
        pf_commit(&drain[1]);
        sh_wait(&drain[1], 0);
      }
    }
    __syncwarp();
    n0 += pc.n;
    ++pieces;
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && warp >= 4 * SG) break;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kCols));
  }
}

// ---------------------------------------------------------------- 16 rows a time, unrounded codes
// The same partials for row tiles of at most 16 rows on mma.sync (m16n8k16), tokens as M, two
// column blocks of 8 rows. Few rows are bound by unpacking the codes, and here they
// meet the tensor cores almost as they are stored:
//   S = sum_g s_g (sum_{d in g} (1024 + n_d) q_d - 1024 sum q_d) + sum_g min_g sum q_d:
//     K's codes are OR-ed into f16 numbers 1024 + n (or + 16 n, against q / 16), one
//     instruction per pair; the accumulator starts at -1024 sum q, exact as the
//     products are; the group's scale multiplies in fp32 afterwards; fp16min's mins
//     are one more product, against sum q_d in f16 high and low parts;
//   O^T += (n V^T) (s_g P)^T: the codes as exact integers, scale times P as two f16 and
//     two products (one f16, rounded apart from P's product with the mins, which the codes'
//     cancels: 2e-4 to 3.9e-4 off in all; the second costs 10 % of fp16min's time and
//     nothing of ref's): of P in f16 (2^-11) for fp16min, whose mins are one more product
//     with that P into an accumulator of its own, of P and the scale in fp32 for ref, whose
//     zero points enter as z sum q_d and as n - z.
// So nothing of K is rounded, and no operand crosses shared memory twice. Against 64
// bits, outliers of ten times the rest among the key channels: fp16min 5e-5 to 1.2e-4 of
// the output in the 2-norm, ref 5e-6 to 1.5e-4 (group 128: the sums of 1024 + n in fp32).
// Two groups
// of four consumer warps take every second tile, 32 tokens a warp.
// Bound by issue and latency of 8 consumer warps an SM (168 registers): 31,680 tokens of
// 8 heads, 32 rows as two row tiles, fp16min 41 us alone, 3,540 warp instructions a tile,
// 40 % of the issue slots, 38 % of the tensor pipe (mma.sync), 21 % of shared memory's
// wavefronts busy; ref (group 32) 47 us, 4,750, 48, 31 and 28 %.
constexpr int kRowsThreads = 320;  // 8 consumer warps, 2 producers
constexpr int kRowsSlots = 6;
constexpr int kRowsPitch = HKV_D + 4;
// P <= 2^4: times a scale it stays below f16's largest for |V| up to 61,000, and P of 2^-14
// is still a normal f16 (with 2^8, and P / 16 for the first, 15,201 tokens of group 128 were
// off by 3.9e-4).
constexpr float kRowsLazy = 4.f;
constexpr int kRowsSmem = kRowsSlots * kShRawBytes + 16 * 256 + 8 * 16 * kRowsPitch * 4;  // raw slots | query fragments | O per warp

template <int FMT, int GROUP>
__global__ void __launch_bounds__(kRowsThreads, 1) shared_rows_kernel(const __grid_constant__ SharedParams p) {
  constexpr int ROWS = 16, NG = HKV_D / GROUP, WPG = 4 / NG, NB = 2, R = kRowsSlots;
  constexpr uint32_t kBlock = block_bytes(FMT, GROUP);
  extern __shared__ __align__(1024) uint8_t sh_raw[];
  __shared__ __align__(8) uint64_t raw_full[R], raw_free[R];
  __shared__ ShGroup s_g[kShMaxGroups + 1];
  __shared__ int s_valid[16];
  __shared__ float s_ps[ROWS][4], s_pb[ROWS][4];                  // per row and 32 dims: sums of q, and of q as multiplied
  __shared__ __align__(8) float s_nb[4][ROWS], s_qs[4][ROWS];    // per group and row: -1024 sum, sum
  __shared__ float s_wm[8][16], s_wl[8][16];                     // per warp and row: m, l
  uint8_t* ring = sh_raw;
  uint4* sQ = reinterpret_cast<uint4*>(ring + R * kShRawBytes);  // [ROWS / 8][4][32 lanes]
  float* comb = reinterpret_cast<float*>(ring + R * kShRawBytes + ROWS * 256);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  if (t == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_free[i], 4);
    }
    fence_barrier_init();
  }
  griddep_launch_dependents();  // the own part may start beside this grid
  if (warp == 0) sh_schedule(p, s_g);
  __syncthreads();
  const int total = s_g[p.P].step;
  int at = sh_cut(total, p.C, blockIdx.x);
  const int end = sh_cut(total, p.C, blockIdx.x + 1);
  uint32_t n0 = 0;  // tiles of the CTA before this piece

  if (warp >= 8) {
    // ---------------- producers: the tiles of the warp's parity ----------------
    const int par = warp - 8;
    bool ok = true;
    uint32_t last = 0;  // behind the last tile issued
    while (ok) {
      const ShPiece pc = sh_next(p, s_g, at, end);
      if (pc.n == 0) break;
      const int u = pc.g * p.Hkv + pc.h, len = s_g[pc.g].len;
      int64_t ids = -1;
      int i = 0;
      for (int j = (n0 ^ par) & 1; j < pc.n; j += 2, ++i) {
        const uint32_t n = n0 + j, slot = n % R;
        const int tok = (pc.t0 + j) * HKV_BLOCK_TOKENS;
        if ((i & 31) == 0) ids = j + 2 * lane < pc.n ? store_page(p.prefix, u, tok + 2 * lane * HKV_BLOCK_TOKENS) : -1;
        const int64_t page = __shfl_sync(0xffffffffu, ids, i & 31);
        if (n >= R && !__all_sync(0xffffffffu, mbar_wait(&raw_free[slot], (n / R - 1) & 1))) {
          ok = false;
          break;
        }
        if (lane == 0) {
          s_valid[n & 15] = page >= 0 ? min(HKV_BLOCK_TOKENS, len - tok) : 0;
          if (page >= 0) {
            const uint8_t* src = static_cast<const uint8_t*>(p.prefix.pages) + page * p.prefix.page_stride +
                                 (int64_t)((tok % p.prefix.page_tokens) / HKV_BLOCK_TOKENS) * kBlock;
            mbar_arrive_expect_tx(&raw_full[slot], kBlock);
            bulk_g2s(ring + slot * kShRawBytes, src, kBlock, &raw_full[slot]);
          } else {  // no such page: the tile counts as hidden
            hkv_flag_error(HKV_DEVERR_BAD_PAGE);
            mbar_arrive(&raw_full[slot]);
          }
        }
        __syncwarp();
        last = n + 1;
      }
      n0 += pc.n;
    }
    // every copy this warp issued lands before the CTA ends (its parity's slots: R is even)
    static_assert(R % 2 == 0, "a slot belongs to one producer");
    for (uint32_t n = last > R ? last - R : 0; n < last; ++n)
      if ((n & 1) == (uint32_t)par) mbar_wait(&raw_full[n % R], (n / R) & 1);
    return;
  }

  // ---------------- consumers ----------------
  const int grp = warp >> 2, wg = warp & 3, r = lane >> 2, j4 = lane & 3, t0 = 32 * wg;
  const float qs = p.qscale;
  bool ok = true;
  while (ok) {
    const ShPiece pc = sh_next(p, s_g, at, end);
    if (pc.n == 0) break;
    const int rows = (p.start[pc.g + 1] - p.start[pc.g]) * p.G - pc.rt * ROWS;
    // query fragments: block b, word w, lane (r, j4): q of row 8 b + r at dims 32 w + 2 j4 + {0, 1},
    // (+ {8, 9}) / 16, + {16, 17}, (+ {24, 25}) / 16; sums of 32 dims beside them
    {
      const int c = warp, b = c >> 2, w = c & 3, n = 8 * b + r;
      uint32_t v[4] = {0u, 0u, 0u, 0u};
      if (n < rows) {
        const int row = pc.rt * ROWS + n, sq = row / p.G;
        const int64_t base = (int64_t)(p.start[pc.g] + sq) * p.q_sb + (int64_t)(pc.h * p.G + row - sq * p.G) * p.q_sh + 32 * w + 2 * j4;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = sh_q2(p, base + 8 * e);
      }
      float ps = 0.f, pb = 0.f;
      uint32_t f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float up = e & 1 ? 16.f : 1.f;
        f[e] = e & 1 ? hmul2(v[e], 0x2C002C00u) : v[e];  // / 16
        const float2 v2 = __half22float2(u2h(f[e]));
        const float sum = v2.x + v2.y;
        pb += sum;
        ps += up * sum;
      }
      sQ[c * 32 + lane] = make_uint4(f[0], f[1], f[2], f[3]);
#pragma unroll
      for (int k = 1; k < 4; k <<= 1) {
        ps += __shfl_xor_sync(0xffffffffu, ps, k);
        pb += __shfl_xor_sync(0xffffffffu, pb, k);
      }
      if (j4 == 0) s_ps[n][w] = ps, s_pb[n][w] = pb;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    for (int c = t; c < NG * ROWS; c += 256) {
      const int g = c / ROWS, n = c - g * ROWS;
      float a = 0.f, b = 0.f;
      for (int w = g * WPG; w < (g + 1) * WPG; ++w) a += s_ps[n][w], b += s_pb[n][w];
      s_qs[g][n] = a;
      s_nb[g][n] = -1024.f * b;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    uint32_t qbias[NB] = {0u, 0u};  // fp16min: sum q_d of the groups, f16 high then low parts, as a B operand
    if constexpr (FMT == HKV_FMT_FP16MIN) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int n = 8 * b + r;
        auto part = [&](int i) -> uint32_t {  // part i < NG: high of group i, else low of group i - NG
          const float v = i < 2 * NG ? s_qs[i % NG][n] : 0.f;
          const __half hi = __float2half_rn(v);
          return i < 2 * NG ? __half_as_ushort(i < NG ? hi : __float2half_rn(v - __half2float(hi))) : 0u;
        };
        qbias[b] = part(2 * j4) | (part(2 * j4 + 1) << 16);
      }
    }
    float o[NB][8][4], zc[NB][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.f;
      zc[b][0] = zc[b][1] = zc[b][2] = zc[b][3] = l[b][0] = l[b][1] = 0.f;
      m[b][0] = m[b][1] = -1.0e30f;
    }
    for (int j = (n0 ^ grp) & 1; j < pc.n; j += 2) {
      const uint32_t n = n0 + j, slot = n % R;
      if (!__all_sync(0xffffffffu, mbar_wait(&raw_full[slot], (n / R) & 1))) {
        ok = false;
        break;
      }
      const uint8_t* blk = ring + slot * kShRawBytes;
      const uint8_t* meta = blk + HKV_META_OFF;
      const int nv = s_valid[n & 15] - t0;  // tokens of this warp's 32 in use
      if (nv > 0) {
        // ---- scores x[s][b]: tokens 16 s + r and 16 s + r + 8, rows 2 j4 and 2 j4 + 1 of block b
        uint32_t kw[2][2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 c = *reinterpret_cast<const uint4*>(blk + (t0 + 8 * i + r) * HKV_CODE_BYTES + 16 * j4);
          kw[i >> 1][i & 1][0] = c.x, kw[i >> 1][i & 1][1] = c.y, kw[i >> 1][i & 1][2] = c.z, kw[i >> 1][i & 1][3] = c.w;
        }
        float sc[2][2][NG], x[2][NB][4];
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          const int tk = t0 + 16 * s2;
#pragma unroll
          for (int b = 0; b < NB; ++b) x[s2][b][0] = x[s2][b][1] = x[s2][b][2] = x[s2][b][3] = 0.f;
          if constexpr (FMT == HKV_FMT_FP16MIN) {
            const __half* ks = reinterpret_cast<const __half*>(meta) + (tk + r) * NG;
            ld_row_h<NG>(ks, 0, sc[s2][0]);
            ld_row_h<NG>(ks, 8, sc[s2][1]);
            // mins of tokens r and r + 8, groups (2 j4, 2 j4 + 1) mod NG, against qbias
            const uint8_t* km = meta + 256 * NG + tk * NG * 2;
            uint32_t m0 = 0u, m1 = 0u;
            if constexpr (NG == 4) {
              m0 = reinterpret_cast<const uint32_t*>(km)[2 * r + (j4 & 1)];
              m1 = reinterpret_cast<const uint32_t*>(km)[2 * (r + 8) + (j4 & 1)];
            } else if constexpr (NG == 2) {
              if (j4 < 2) m0 = reinterpret_cast<const uint32_t*>(km)[r], m1 = reinterpret_cast<const uint32_t*>(km)[r + 8];
            } else if (j4 == 0) {
              m0 = reinterpret_cast<const uint16_t*>(km)[r] * 0x10001u;
              m1 = reinterpret_cast<const uint16_t*>(km)[r + 8] * 0x10001u;
            }
            const uint32_t ab[4] = {m0, m1, 0u, 0u};
#pragma unroll
            for (int b = 0; b < NB; ++b) mma16816<__half>(x[s2][b], ab, qbias[b], 0u);
          } else {
            const float* ks = reinterpret_cast<const float*>(meta) + (tk + r) * NG;
            ld_row<NG>(ks, 0, sc[s2][0]);
            ld_row<NG>(ks, 8, sc[s2][1]);
          }
        }
        float c[2][NB][4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int g = w / WPG;
          uint32_t a0[2][4], a1[2][4];
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            const uint32_t wa = kw[s2][0][w], wb = kw[s2][1][w], wa8 = wa >> 8, wb8 = wb >> 8;
            a0[s2][0] = biased1(wa), a0[s2][1] = biased1(wb), a0[s2][2] = biased16(wa), a0[s2][3] = biased16(wb);
            a1[s2][0] = biased1(wa8), a1[s2][1] = biased1(wb8), a1[s2][2] = biased16(wa8), a1[s2][3] = biased16(wb8);
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint4 f = sQ[(b * 4 + w) * 32 + lane];
            if (w % WPG == 0) {
              const float2 nb = *reinterpret_cast<const float2*>(&s_nb[g][8 * b + 2 * j4]);
              const float ci[4] = {nb.x, nb.y, nb.x, nb.y};
              mma16816_c(c[0][b], a0[0], f.x, f.y, ci);
              mma16816_c(c[1][b], a0[1], f.x, f.y, ci);
            } else {
              mma16816<__half>(c[0][b], a0[0], f.x, f.y);
              mma16816<__half>(c[1][b], a0[1], f.x, f.y);
            }
            mma16816<__half>(c[0][b], a1[0], f.z, f.w);
            mma16816<__half>(c[1][b], a1[1], f.z, f.w);
            if (w % WPG == WPG - 1) {
#pragma unroll
              for (int s2 = 0; s2 < 2; ++s2) {
                float *xx = x[s2][b], *cc = c[s2][b];
                if constexpr (FMT == HKV_FMT_REF) {  // minus the zero points' share
                  const float2 q2 = *reinterpret_cast<const float2*>(&s_qs[g][8 * b + 2 * j4]);
                  const uint8_t* kz = meta + 1024 * NG + (t0 + 16 * s2 + r) * NG + g;
                  const float za = -(float)kz[0], zb = -(float)kz[8 * NG];
                  cc[0] = fmaf(za, q2.x, cc[0]), cc[1] = fmaf(za, q2.y, cc[1]);
                  cc[2] = fmaf(zb, q2.x, cc[2]), cc[3] = fmaf(zb, q2.y, cc[3]);
                }
                const float2 lo = __ffma2_rn(make_float2(sc[s2][0][g], sc[s2][0][g]), make_float2(cc[0], cc[1]), make_float2(xx[0], xx[1]));
                const float2 hi = __ffma2_rn(make_float2(sc[s2][1][g], sc[s2][1][g]), make_float2(cc[2], cc[3]), make_float2(xx[2], xx[3]));
                xx[0] = lo.x, xx[1] = lo.y, xx[2] = hi.x, xx[3] = hi.y;
              }
            }
          }
        }
        // ---- softmax: the warp's own running max, moved when a score beats it by 2^4
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float* xx = x[s2][b];
            const float2 lo = __fmul2_rn(make_float2(xx[0], xx[1]), make_float2(qs, qs)), hi = __fmul2_rn(make_float2(xx[2], xx[3]), make_float2(qs, qs));
            xx[0] = lo.x, xx[1] = lo.y, xx[2] = hi.x, xx[3] = hi.y;
          }
        if (nv < 32) {  // the prefix ends in here
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (16 * s2 + r + 4 * (i & 2) >= nv) x[s2][b][i] = -INFINITY;
        }
        float top[NB][2];
        bool need = false;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[b][e] = fmax3(fmaxf(x[0][b][e], x[0][b][e + 2]), x[1][b][e], x[1][b][e + 2]);
            need |= top[b][e] > m[b][e] + kRowsLazy;
          }
        if (__any_sync(0xffffffffu, need)) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = top[b][e];
#pragma unroll
              for (int k = 4; k < 32; k <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, k));
              const float nm = fmaxf(m[b][e], v), a = fast_exp2(m[b][e] - nm);
              m[b][e] = nm;
              l[b][e] *= a;
#pragma unroll
              for (int i = 0; i < 8; ++i) o[b][i][e] *= a, o[b][i][e + 2] *= a;
              zc[b][e] *= a, zc[b][e + 2] *= a;
            }
        }
        // x becomes P; fp16min: in f16, transposed: row r, tokens 2 j4, 2 j4 + 1 (+ 8)
        uint32_t pt[2][NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float m0 = m[b][0], m1 = m[b][1];
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            float* xx = x[s2][b];
            xx[0] = fast_exp2(xx[0] - m0), xx[1] = fast_exp2(xx[1] - m1);
            xx[2] = fast_exp2(xx[2] - m0), xx[3] = fast_exp2(xx[3] - m1);
            l[b][0] += xx[0] + xx[2];
            l[b][1] += xx[1] + xx[3];
            if constexpr (FMT == HKV_FMT_FP16MIN) {
              pt[s2][b][0] = movmatrix_t(pack2<__half>(xx[0], xx[1]));
              pt[s2][b][1] = movmatrix_t(pack2<__half>(xx[2], xx[3]));
            }
          }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          const int q0 = (t0 + 16 * s2) / 2, left = nv - 16 * s2;  // the subtile's first pair; its tokens in use
          uint32_t vs[2][NG], vz[2][NG];  // pairs j4 and 4 + j4: fp16min's scales; ref's zero points
          float vf[2][NG];                // ref: scales of tokens r and r + 8
          uint32_t zmin[2] = {0u, 0u};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int q = q0 + 4 * e + j4;
            if constexpr (FMT == HKV_FMT_FP16MIN) {
              ld_row_u<NG>(reinterpret_cast<const uint32_t*>(meta + 512 * NG), q, vs[e]);
              zmin[e] = r < NG ? reinterpret_cast<const uint32_t*>(meta + 768 * NG)[q * NG + r] : 0u;
            } else {
              ld_row<NG>(reinterpret_cast<const float*>(meta + 512 * NG), 2 * q0 + 8 * e + r, vf[e]);
              const uint8_t* zp = meta + 1152 * NG + 2 * q * NG;
#pragma unroll
              for (int g = 0; g < NG; ++g) vz[e][g] = (uint32_t)zp[g] | ((uint32_t)zp[NG + g] << 16);
            }
          }
          if (left < 16) {  // unused tokens' metadata may be any bits: P = 0 has to meet 0
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int tk = 8 * e + 2 * j4;
              const uint32_t keep = (tk < left ? 0x0000FFFFu : 0u) | (tk + 1 < left ? 0xFFFF0000u : 0u);
              zmin[e] &= keep;
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                if constexpr (FMT == HKV_FMT_FP16MIN) vs[e][g] &= keep;
                else vf[e][g] = 8 * e + r < left ? vf[e][g] : 0.f;
              }
            }
          }
          if constexpr (FMT == HKV_FMT_FP16MIN) {
            const uint32_t ab[4] = {zmin[0], 0u, zmin[1], 0u};
#pragma unroll
            for (int b = 0; b < NB; ++b) mma16816<__half>(zc[b], ab, pt[s2][b][0], pt[s2][b][1]);
          }
          uint32_t vw[2][4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint4 c4 = *reinterpret_cast<const uint4*>(blk + HKV_V_CODES_OFF + v_chunk_off(q0 + 4 * e + j4, r));
            vw[e][0] = c4.x, vw[e][1] = c4.y, vw[e][2] = c4.z, vw[e][3] = c4.w;
          }
          // the codes' other operand, P times the group's scale, as two f16, the second what the
          // first leaves: of P as it meets the mins (fp16min), of the fp32 product (ref)
          uint32_t ph[NB][2], pl[NB][2];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int g = k / WPG;
            if (k % WPG == 0) {
#pragma unroll
              for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  if constexpr (FMT == HKV_FMT_FP16MIN) {
                    ph[b][e] = hmul2(pt[s2][b][e], vs[e][g]);
                    pl[b][e] = h2u(__hfma2(u2h(pt[s2][b][e]), u2h(vs[e][g]), __hneg2(u2h(ph[b][e]))));
                  } else {
                    const float2 y = __fmul2_rn(make_float2(x[s2][b][2 * e], x[s2][b][2 * e + 1]), make_float2(vf[e][g], vf[e][g]));
                    const uint32_t hi = pack2<__half>(y.x, y.y);
                    const float2 z = __half22float2(u2h(hi));
                    ph[b][e] = movmatrix_t(hi);
                    pl[b][e] = movmatrix_t(pack2<__half>(y.x - z.x, y.y - z.y));
                  }
                }
            }
            uint32_t ha[4], hb[4];
            if constexpr (FMT == HKV_FMT_REF) {  // 1024 + z and -64 - z in f16 are one addition to the bits
              nib8_to_h2_z(vw[0][k], 0x64006400u + vz[0][g], 0xD400D400u + 16u * vz[0][g], ha);
              nib8_to_h2_z(vw[1][k], 0x64006400u + vz[1][g], 0xD400D400u + 16u * vz[1][g], hb);
            } else {
              nib8_to_h2(vw[0][k], ha);
              nib8_to_h2(vw[1][k], hb);
            }
            const uint32_t a0[4] = {ha[0], ha[1], hb[0], hb[1]}, a1[4] = {ha[2], ha[3], hb[2], hb[3]};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              mma16816<__half>(o[b][2 * k], a0, ph[b][0], ph[b][1]);
              mma16816<__half>(o[b][2 * k + 1], a1, ph[b][0], ph[b][1]);
              mma16816<__half>(o[b][2 * k], a0, pl[b][0], pl[b][1]);
              mma16816<__half>(o[b][2 * k + 1], a1, pl[b][0], pl[b][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_free[slot]);
    }
    n0 += pc.n;
    // ---- the piece's partial: the warps' O, m, l joined through shared memory
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], k);
        if (r == 0) s_wm[warp][8 * b + 2 * j4 + e] = m[b][e], s_wl[warp][8 * b + 2 * j4 + e] = l[b][e];
        float z[NG];  // fp16min: row g of the mins' product is in lane 4 g + j4
#pragma unroll
        for (int g = 0; g < NG; ++g) z[g] = FMT == HKV_FMT_FP16MIN ? __shfl_sync(0xffffffffu, zc[b][e], 4 * g + j4) : 0.f;
        float* dst = comb + (warp * 16 + 8 * b + 2 * j4 + e) * kRowsPitch + r;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float zz = z[16 * i / GROUP];
          dst[16 * i] = o[b][i][e] + zz;
          dst[16 * i + 8] = o[b][i][e + 2] + zz;
        }
      }
    }
    if (!bar_and(1, 256, ok)) break;
    const int64_t id = (int64_t)(blockIdx.x + pc.unit) * ROWS;
    for (int c = t; c < ROWS * 32; c += 256) {  // (row, 4 dims)
      const int n = c >> 5, d = 4 * (c & 31);
      float M = -1.0e30f, L = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) M = fmaxf(M, s_wm[w][n]);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float x = fast_exp2(s_wm[w][n] - M);
        const float4 v = *reinterpret_cast<const float4*>(comb + (w * 16 + n) * kRowsPitch + d);
        L += x * s_wl[w][n];
        a = make_float4(a.x + x * v.x, a.y + x * v.y, a.z + x * v.z, a.w + x * v.w);
      }
      if (n < rows) {
        *reinterpret_cast<float4*>(p.part_o + (id + n) * HKV_D + d) = a;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (id + n) * 2) = make_float2(M, L);
      }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the shared tables and areas are free again
  }
}

// out[b][hq] from the partials of the row's pieces and of its own tokens:
// sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i. Four warps per row, each a quarter
// of the partials (lane = dims 4 lane .. 4 lane + 3), all (m, l) and then several
// O loaded at once: the launch is a few round trips to L2, not one per partial.
__global__ void __launch_bounds__(128) shared_merge_kernel(const __grid_constant__ SharedParams p) {
  __shared__ ShGroup s_g[kShMaxGroups + 1];
  __shared__ float4 s_o[4][32];
  __shared__ float2 s_ml[4];
  if (threadIdx.x < 32) sh_schedule(p, s_g);
  __syncthreads();
  const int Hq = p.Hkv * p.G, row = blockIdx.x, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int b = row / Hq, hq = row - b * Hq, h = hq / p.G;
  const int total = s_g[p.P].step;
  int g = 0;
  for (int hi = p.P; g < hi;) {  // the first group that ends behind b
    const int mid = (g + hi) >> 1;
    if (p.start[mid + 1] > b) hi = mid;
    else g = mid + 1;
  }
  int c0 = 0, c1 = -1, unit = 0, n = 0;
  if (g < p.P && p.start[g] <= b && s_g[g + 1].step > s_g[g].step) {
    const int units = s_g[g + 1].unit - s_g[g].unit, per = (s_g[g + 1].step - s_g[g].step) / units, rts = units / p.Hkv;
    const int r = (b - p.start[g]) * p.G + hq - h * p.G, rt = r / p.N, u = h * rts + rt;
    n = r - rt * p.N;
    unit = s_g[g].unit + u;
    const int first = s_g[g].step + u * per + kShCharge, last = first + per - kShCharge - 1;
    auto cta = [&](int step) {
      int c = (int)((int64_t)step * p.C / total);
      while (c + 1 < p.C && sh_cut(total, p.C, c + 1) <= step) ++c;
      while (c > 0 && sh_cut(total, p.C, c) > step) --c;
      return c;
    };
    c0 = cta(first);
    c1 = cta(last);
  }
  // partial k: the own part (k = 0, when there is one), then the streams of the CTAs c0 .. c1
  const int own = p.own_o ? 1 : 0, ns = p.ns, parts = own + (c1 - c0 + 1) * ns;
  float M = -1.0e30f, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = w; k0 < parts; k0 += 128) {  // up to 32 partials of this warp: k0, k0 + 4, ...
    const int k = k0 + 4 * lane, c = c0 + (k - own) / ns;
    float2 ml = make_float2(-1.0e30f, 0.f);
    const float* src = nullptr;
    if (k < own) {
      ml = *reinterpret_cast<const float2*>(p.own_ml + (int64_t)row * 2);
      src = p.own_o + (int64_t)row * HKV_D;
    } else if (k < parts && sh_cut(total, p.C, c) < sh_cut(total, p.C, c + 1)) {  // else: more CTAs than steps
      const int64_t id = ((int64_t)(c + unit) * ns + (k - own) % ns) * p.N + n;
      ml = *reinterpret_cast<const float2*>(p.part_ml + id * 2);
      src = p.part_o + id * HKV_D;
    }
    if (ml.y == 0.f) ml.x = -1.0e30f, src = nullptr;  // saw nothing
    float nm = fmaxf(M, ml.x);
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, x));
    const float a = fast_exp2(M - nm), wt = src ? fast_exp2(ml.x - nm) : 0.f;
    float l = src ? ml.y * wt : 0.f;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    M = nm;
    L = L * a + l;
    acc = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
    const int m = min(32, (parts - k0 + 3) / 4);
#pragma unroll 4
    for (int i = 0; i < m; ++i) {
      const float* o = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), i));
      const float x = __shfl_sync(0xffffffffu, wt, i);
      if (o) {
        const float4 v = *reinterpret_cast<const float4*>(o + 4 * lane);
        acc = make_float4(acc.x + v.x * x, acc.y + v.y * x, acc.z + v.z * x, acc.w + v.w * x);
      }
    }
  }
  s_o[w][lane] = acc;
  if (lane == 0) s_ml[w] = make_float2(M, L);
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) M = fmaxf(M, s_ml[i].x);
  L = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = fast_exp2(s_ml[i].x - M);
    const float4 v = s_o[i][lane];
    L += s_ml[i].y * x;
    acc = make_float4(acc.x + v.x * x, acc.y + v.y * x, acc.z + v.z * x, acc.w + v.w * x);
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;  // a NaN stays one
  const int64_t ob = (int64_t)b * p.out_sb + (int64_t)hq * p.out_sh + 4 * lane;
  const float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) store_any(p.out, p.out_dtype, ob + i, v[i] * inv);
}

}  // namespace hkv
