// Cross attention to an encoder's states of another length (gfx950), for
// bf16, fp16 and fp32 tensors: forward, backward and the one-token form.
//
// Per sample b and key head g (the G = H / Hk query heads that share it are
// rows of one matrix: row r is token r / G, head g G + r % G):
//   P = softmax_j(scale Q K^T) over the kept states j < kv_lens[b], mask[b][j]
//   O = P V;  a row without kept states, or past q_lens[b], is zero.
//   delta_i = dO_i . O_i;  dP = dO V^T;  dS = P (dP - delta)
//   dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO
// One pass over the states with a running maximum and sum; the matrix of
// scores never leaves the registers.
//
// Every kernel has one side that a wave owns (32 rows, or in xattn_dkv 32
// states, one per lane) and one that is streamed through LDS.  The first
// product puts the owned side on the MFMA columns, S^T = K Q^T, so one lane
// holds one row's scores: maximum and sum are lane-local plus one exchange
// with the other half of the wave, and the accumulator as it stands is the B
// operand of the second product (O^T = V^T P^T, dQ^T = K^T dS^T,
// dV^T = dO^T P, dK^T = Q^T dS), whose k axis runs in the accumulator's row
// order; its A operand is read from LDS transposed in that order.
//
// fp32 runs on v_mfma_f32_32x32x2_f32 (every product and sum in 32 bits).
// bf16 / fp16 round P and dS to the type as MFMA operands (2^-9 / 2^-12
// relative, of the size of the one rounding of the result); sums, statistics
// and accumulators are fp32.
//
// Masked states never reach a product: their rows of K and V are written to
// LDS as zeros (NaN or infinity there stays there) and their scores are -inf.
#pragma once
#include <type_traits>

#include "tgfr_common.h"

namespace tgfr {

constexpr float LOG2E_X = 1.4426950408889634f;

// element strides of a [B][T][H][D] tensor with unit stride over D
struct XView {
  void* p;
  long long sb, st, sh;
};

struct XArgs {
  XView q, k, v, o, dout, dq, dk, dv;
  const int* q_lens;     // [B] or NULL
  const int* kv_lens;    // [B] or NULL
  const uint8_t* mask;   // [B][Tk], row stride mask_sb; nonzero: attended to; or NULL
  long long mask_sb;
  float* lse;            // [B Hk][R]: log2 of the row's sum, in the log2 domain; +inf: none
  float* delta;          // [B Hk][R]
  float* amax;           // [B Hk][R] largest |dO| of the row (fp16 only)
  float* part;           // partial results of the splits
  float* part_ml;        // forward: [split][B Hk][R][2] maximum and sum
  int B, Tq, Tk, H, Hk, G, D, R;   // R = Tq G
  int splits, tiles;
  float scale;
};

struct XBf16 {
  static constexpr int TYPE = 0, ES = 2;
  using elem = uint16_t;
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(a), as_bf8(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pk(float a, float b) { return pk_bf16(a, b); }
  static __device__ __forceinline__ float val(uint16_t u) { return bf_val(u); }
  static __device__ __forceinline__ uint16_t bits(float x) { return bf_bits(x); }
};
struct XF16 {
  static constexpr int TYPE = 2, ES = 2;
  using elem = uint16_t;
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pk(float a, float b) {
    return pk_lowp<MODE_F16>(a, b);
  }
  static __device__ __forceinline__ float val(uint16_t u) {
    return (float)__builtin_bit_cast(_Float16, u);
  }
  static __device__ __forceinline__ uint16_t bits(float x) { return f16_bits(x); }
};
struct XF32 {
  static constexpr int TYPE = 1, ES = 4;
  using elem = float;
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float val(float x) { return x; }
  static __device__ __forceinline__ float bits(float x) { return x; }
};

// 16 bytes at an address aligned to the element only (gfx950 reads and writes
// global memory at any alignment)
typedef u32x4 u32x4_u __attribute__((aligned(2)));

__device__ __forceinline__ uint4 zero16() { return make_uint4(0, 0, 0, 0); }

// Chunk `ch` (16 bytes) of a row of D elements; elements past D are zero.
template <class T>
__device__ __forceinline__ uint4 ld_chunk(const typename T::elem* row, int ch, int D) {
  constexpr int E = 16 / T::ES;
  const int d0 = ch * E;
  if (d0 + E <= D)
    return __builtin_bit_cast(uint4, (u32x4) * (const u32x4_u*)(row + d0));
  typename T::elem e[E];
#pragma unroll
  for (int i = 0; i < E; ++i) e[i] = d0 + i < D ? row[d0 + i] : (typename T::elem)0;
  return __builtin_bit_cast(uint4, e);
}
template <class T>
__device__ __forceinline__ void st_chunk(typename T::elem* row, int ch, int D, uint4 v) {
  constexpr int E = 16 / T::ES;
  const int d0 = ch * E;
  if (d0 + E <= D) {
    *(u32x4_u*)(row + d0) = __builtin_bit_cast(u32x4, v);
    return;
  }
  typename T::elem e[E];
  __builtin_memcpy(e, &v, 16);
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (d0 + i < D) row[d0 + i] = e[i];
}

// LDS image of rows of DP elements: 16-byte chunk c of row r lies at chunk
// c ^ f(r).  Free of bank conflicts for both ways of reading: one logical
// chunk of 16 consecutive rows (f is one-to-one on r mod 16 together with the
// row's place in its 256-byte line), and four consecutive rows of the chunks
// of 32 columns, transposed.
template <class T, int DP>
struct Img {
  static constexpr int ROWB = DP * T::ES;
  static constexpr int CPR = ROWB / 16;
  static constexpr int E = 16 / T::ES;
  static constexpr int NC = CPR / 2;            // MFMA steps over D
  static constexpr int NPF = T::ES == 2 ? 2 : 4;   // B operands of 32 accumulator rows
  static constexpr int bytes(int rows) { return rows * ROWB; }

  static __device__ __forceinline__ int f(int r) {
    if constexpr (CPR >= 16)
      return 4 * (r & 3) + ((r >> 2) & 3);
    else
      return 4 * ((r >> 1) & 1) + ((r >> 2) & 3);
  }
  static __device__ __forceinline__ uint32_t at(int r, int ch) {
    return (uint32_t)(r * ROWB + ((ch ^ f(r)) << 4));
  }
  // A operand, row r0 + lane % 32 (r0 a multiple of 16), MFMA step j
  static __device__ __forceinline__ uint4 rm(uint32_t base, int r0, int j, int lane) {
    const int r = lane & 31;
    return lds_ld16(base + r0 * ROWB + r * ROWB + (((2 * j + (lane >> 5)) ^ f(r)) << 4));
  }
  // A operand, column 32 db + lane % 32 at the rows r0 + acc_row order of
  // B operand c (r0 a multiple of 32)
  static __device__ __forceinline__ uint4 tr(uint32_t base, int r0, int c, int db, int lane) {
    if constexpr (T::ES == 2) {
      const int i = lane & 15, g = lane >> 4, h = g >> 1, q = i >> 2;
      const int ch = 4 * db + 2 * (g & 1) + ((i >> 1) & 1), in = 8 * (i & 1);
      s16x4 v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * e + 4 * h + q;          // + 16 c + r0: f is the same
        v[e] = lds_tr4(base + (r0 + 16 * c) * ROWB + r * ROWB + ((ch ^ f(r)) << 4) + in);
      }
      return __builtin_bit_cast(uint4, join_tr(v[0], v[1]));
    } else {
      const int col = 32 * db + (lane & 31), h = lane >> 5;
      uint4 v;
      uint32_t* o = (uint32_t*)&v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 8 * (c & 1) + 4 * h + e;
        o[e] = __float_as_uint(lds_ldf(base + (r0 + 16 * (c >> 1)) * ROWB + r * ROWB +
                                       (((col >> 2) ^ f(r)) << 4) + 4 * (col & 3)));
      }
      return v;
    }
  }
  // B operand c of 32 accumulator rows
  static __device__ __forceinline__ uint4 pack(const f32x16& s, int c) {
    if constexpr (T::ES == 2)
      return make_uint4(T::pk(s[8 * c], s[8 * c + 1]), T::pk(s[8 * c + 2], s[8 * c + 3]),
                        T::pk(s[8 * c + 4], s[8 * c + 5]), T::pk(s[8 * c + 6], s[8 * c + 7]));
    else
      return make_uint4(__float_as_uint(s[4 * c]), __float_as_uint(s[4 * c + 1]),
                        __float_as_uint(s[4 * c + 2]), __float_as_uint(s[4 * c + 3]));
  }
};

// A tile of ROWS rows in flight from global memory to LDS, held in registers.
template <class T, int DP, int ROWS, int NT>
struct Stage {
  using I = Img<T, DP>;
  static constexpr int N = ROWS * I::CPR / NT;
  static_assert(ROWS * I::CPR % NT == 0, "whole chunks per thread");
  uint4 r[N];

  // row(i): pointer to row i of the tile, or NULL for zeros
  template <class Row>
  __device__ __forceinline__ void load(Row row, int D) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = threadIdx.x + NT * n;
      const typename T::elem* p = row(idx / I::CPR);
      const int ch = idx % I::CPR;
      r[n] = p && ch * I::E < D ? ld_chunk<T>(p, ch, D) : zero16();
    }
  }
  __device__ __forceinline__ void store(uint32_t base) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = threadIdx.x + NT * n;
      lds_st16(base + I::at(idx / I::CPR, idx % I::CPR), r[n]);
    }
  }
  template <int W>
  __device__ __forceinline__ void store_kept(uint32_t base, const uint64_t (&keep)[W]) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = threadIdx.x + NT * n, row = idx / I::CPR;
      const bool k = (keep[W == 1 ? 0 : row >> 6] >> (row & 63)) & 1;
      lds_st16(base + I::at(row, idx % I::CPR), k ? r[n] : zero16());
    }
  }
};

// ------------------------------------------------------------ shared parts ---
// The block's work: sample, key head, tile of rows (or states), split.
struct XWork {
  int b, g, bh, tile, split;
};
__device__ __forceinline__ XWork x_work(const XArgs& a) {
  // consecutive work shares K and V (or Q and dO), and so one XCD's L2
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  XWork w;
  w.tile = id % a.tiles;
  const int rest = id / a.tiles;
  w.bh = rest % (a.B * a.Hk);
  w.split = rest / (a.B * a.Hk);
  w.b = w.bh / a.Hk;
  w.g = w.bh % a.Hk;
  return w;
}
__device__ __forceinline__ int x_len(const int* lens, int b, int T) {
  return lens ? min(max(lens[b], 0), T) : T;
}
template <class E>
__device__ __forceinline__ E* x_row(const XView& v, int b, int g, int G, int r) {
  const int t = G == 1 ? r : (int)((unsigned)r / (unsigned)G);
  return (E*)v.p + b * v.sb + t * v.st + (long long)(g * G + (r - t * G)) * v.sh;
}
template <class E>
__device__ __forceinline__ E* x_key(const XView& v, int b, int g, int j) {
  return (E*)v.p + b * v.sb + j * v.st + g * v.sh;
}
// [first, last) of a split's share of n items in whole tiles
__device__ __forceinline__ void x_share(int n, int tile, int splits, int split, int& lo, int& hi) {
  const int nt = (n + tile - 1) / tile, per = (nt + splits - 1) / splits;
  lo = min(n, split * per * tile);
  hi = min(n, (split + 1) * per * tile);
}
// which of the tile's states are attended to, one bit each, equal in all waves
template <int KT>
struct Keep {
  static constexpr int W = (KT + 63) / 64;
  uint8_t m[W];
  __device__ __forceinline__ void load(const uint8_t* mask, int k0, int len, int lane) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int j = k0 + 64 * w + lane;
      m[w] = j < len ? (mask ? mask[j] : 1) : 0;
    }
  }
  __device__ __forceinline__ void bits(uint64_t (&keep)[W]) const {
#pragma unroll
    for (int w = 0; w < W; ++w) keep[w] = __ballot(m[w] != 0);
  }
};

// Writes WR * 32 rows of DP accumulated values (acc[db][q]: column
// 32 db + acc_row(q, h) of the wave's row lane % 32), summed over the WS waves
// that share the rows, times mul, through LDS at `lb`, so that whole rows are
// written.  dst(row) is the row's place, or NULL; tid: the thread's number
// among the 64 WR WS that write these rows.  All waves of the block call it.
template <class T, int DP, int WR, int WS, class Dst>
__device__ __forceinline__ void x_store(const f32x16 (&acc)[DP / 32], float mul, bool zero, int D,
                                        int tid, uint32_t lb, Dst dst) {
  using I = Img<T, DP>;
  const int lane = tid % 64, wave = tid / 64, wr = wave % WR, ws = wave / WR;
  const int r = lane & 31, h = lane >> 5;
  __syncthreads();
  if constexpr (WS == 1) {
    const uint32_t base = lb + wave * I::bytes(32);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = zero ? 0.f : acc[db][4 * k + e] * mul;
        const int d = 32 * db + 8 * k + 4 * h;
        const uint32_t p = base + I::at(r, d / I::E);
        if constexpr (T::ES == 2)
          lds_st8(p + 2 * (d % 8), make_uint2(T::pk(v[0], v[1]), T::pk(v[2], v[3])));
        else
          lds_st16(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]),
                                 __float_as_uint(v[2]), __float_as_uint(v[3])));
      }
    __syncthreads();
    for (int idx = lane; idx < 32 * I::CPR; idx += 64) {
      const int row = idx / I::CPR, ch = idx % I::CPR;
      typename T::elem* p = ch * I::E < D ? dst(32 * wave + row) : nullptr;
      if (p) st_chunk<T>(p, ch, D, lds_ld16(base + I::at(row, ch)));
    }
  } else {
    using F = Img<XF32, DP>;
    const uint32_t base = lb + (ws * WR + wr) * F::bytes(32);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = zero ? 0.f : acc[db][4 * k + e] * mul;
        lds_st16(base + F::at(r, 8 * db + 2 * k + h),
                 make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                            __float_as_uint(v[3])));
      }
    __syncthreads();
    for (int idx = tid; idx < WR * 32 * I::CPR; idx += 64 * WR * WS) {
      const int row = idx / I::CPR, ch = idx % I::CPR;
      typename T::elem* p = ch * I::E < D ? dst(row) : nullptr;
      if (!p) continue;
      float s[I::E] = {};
      for (int w = 0; w < WS; ++w)
#pragma unroll
        for (int c = 0; c < I::E / 4; ++c) {
          const uint4 u = lds_ld16(lb + w * F::bytes(WR * 32) + F::at(row, ch * (I::E / 4) + c));
          s[4 * c] += __uint_as_float(u.x);
          s[4 * c + 1] += __uint_as_float(u.y);
          s[4 * c + 2] += __uint_as_float(u.z);
          s[4 * c + 3] += __uint_as_float(u.w);
        }
      uint4 v;
      if constexpr (T::ES == 2)
        v = make_uint4(T::pk(s[0], s[1]), T::pk(s[2], s[3]), T::pk(s[4], s[5]), T::pk(s[6], s[7]));
      else
        v = make_uint4(__float_as_uint(s[0]), __float_as_uint(s[1]), __float_as_uint(s[2]),
                       __float_as_uint(s[3]));
      st_chunk<T>(p, ch, D, v);
    }
  }
}
// LDS that x_store needs
template <class T, int DP, int WR, int WS>
constexpr int x_store_bytes() {
  return WS == 1 ? Img<T, DP>::bytes(32 * WR) : Img<XF32, DP>::bytes(32 * WR * WS);
}
constexpr int x_max(int a, int b) { return a > b ? a : b; }

// ------------------------------------------------------------------ forward ---
// WR waves along the rows (32 each) x WS waves along the states of a tile.
template <class T, int DP, int WR, int WS, int KT>
struct FwdCfg {
  static constexpr int NT = 64 * WR * WS;
  static constexpr int SUB = KT / WS / 32;      // 32-state pieces of a wave per tile
  static constexpr int ML = x_max(2 * Img<T, DP>::bytes(KT), x_store_bytes<T, DP, WR, WS>());
  static constexpr int LDS = ML + (WS > 1 ? 2 * 4 * 32 * WR * WS : 0);
};

template <class T, int DP, int WR, int WS, int KT, int OCC>
__global__ __launch_bounds__(64 * WR * WS, OCC) void xattn_fwd(const XArgs a) {
  using I = Img<T, DP>;
  using C = FwdCfg<T, DP, WR, WS, KT>;
  using E = typename T::elem;
  const XWork w = x_work(a);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wr = wave % WR, ws = wave / WR;
  const int lr = lane & 31, h = lane >> 5;
  const int rows = x_len(a.q_lens, w.b, a.Tq) * a.G;
  const int row0 = w.tile * WR * 32, row = row0 + wr * 32 + lr;
  const int len = row0 < rows ? x_len(a.kv_lens, w.b, a.Tk) : 0;
  int klo, khi;
  x_share(len, KT, a.splits, w.split, klo, khi);
  const uint8_t* mask = a.mask ? a.mask + w.b * a.mask_sb : nullptr;
  const uint32_t LK = 0, LV = I::bytes(KT);
  const float c2 = a.scale * LOG2E_X;

  uint4 qf[I::NC];
  {
    const E* p = row < rows ? x_row<E>(a.q, w.b, w.g, a.G, row) : nullptr;
#pragma unroll
    for (int j = 0; j < I::NC; ++j)
      qf[j] = p && (2 * j + h) * I::E < a.D ? ld_chunk<T>(p, 2 * j + h, a.D) : zero16();
  }
  f32x16 acc[DP / 32] = {};
  float m = -INFINITY, l = 0.f;

  Stage<T, DP, KT, C::NT> sk, sv;
  Keep<KT> kp;
  auto fetch = [&](int k0) {
    kp.load(mask, k0, khi, lane);
    sk.load([&](int r) { return k0 + r < khi ? x_key<E>(a.k, w.b, w.g, k0 + r) : nullptr; }, a.D);
    sv.load([&](int r) { return k0 + r < khi ? x_key<E>(a.v, w.b, w.g, k0 + r) : nullptr; }, a.D);
  };
  if (klo < khi) fetch(klo);
  for (int k0 = klo; k0 < khi; k0 += KT) {
    uint64_t keep[Keep<KT>::W];
    kp.bits(keep);
    __syncthreads();
    sk.store_kept(LK, keep);
    sv.store_kept(LV, keep);
    __syncthreads();
    if (k0 + KT < khi) fetch(k0 + KT);

    f32x16 s[C::SUB];
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < C::SUB; ++u) {
      const int r0 = (ws * C::SUB + u) * 32;
      s[u] = f32x16{};
#pragma unroll
      for (int j = 0; j < I::NC; ++j) s[u] = T::mma(I::rm(LK, r0, j, lane), qf[j], s[u]);
      const uint32_t kb = (uint32_t)(keep[r0 >> 6] >> (r0 & 63));
      if (kb != 0xffffffffu) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[u][e] = (kb >> acc_row(e, h)) & 1 ? s[u][e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[u][e]);
    }
    // log2 domain: exp(scale s - max) = 2^(c2 s - m)
    const float mn = fmaxf(m, xhalf_max(top) * c2);
    const float mu = mn == -INFINITY ? 0.f : mn;      // no kept state so far
    const float al = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    l *= al;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) acc[db] *= al;
#pragma unroll
    for (int u = 0; u < C::SUB; ++u) {
      const int r0 = (ws * C::SUB + u) * 32;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], c2, -mu));
        l += s[u][e];
      }
#pragma unroll
      for (int c = 0; c < I::NPF; ++c) {
        const uint4 p = I::pack(s[u], c);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] = T::mma(I::tr(LV, r0, c, db, lane), p, acc[db]);
      }
    }
  }
  l = xhalf_sum(l);

  float mul = 1.f;
  if constexpr (WS > 1) {       // the waves that share rows agree on the maximum
    const uint32_t ML = C::ML;
    __syncthreads();
    if (h == 0) {
      lds_stf(ML + 4 * ((ws * WR + wr) * 32 + lr), m);
      lds_stf(ML + 4 * ((WS * WR + ws * WR + wr) * 32 + lr), l);
    }
    __syncthreads();
    float mm = -INFINITY, ll = 0.f;
    for (int x = 0; x < WS; ++x) mm = fmaxf(mm, lds_ldf(ML + 4 * ((x * WR + wr) * 32 + lr)));
    const float mu = mm == -INFINITY ? 0.f : mm;
    for (int x = 0; x < WS; ++x)
      ll += lds_ldf(ML + 4 * ((WS * WR + x * WR + wr) * 32 + lr)) *
            __builtin_amdgcn_exp2f(lds_ldf(ML + 4 * ((x * WR + wr) * 32 + lr)) - mu);
    mul = __builtin_amdgcn_exp2f(m - mu);
    m = mm;
    l = ll;
  }
  const bool none = !(row < rows) || m == -INFINITY && l == 0.f;
  const long long at = (long long)w.bh * a.R;
  if (a.splits == 1) {
    if (a.lse && ws == 0 && h == 0 && row < a.R)
      a.lse[at + row] = none ? INFINITY : m + __builtin_amdgcn_logf(l);
    x_store<T, DP, WR, WS>(acc, mul / l, none, a.D, threadIdx.x, 0, [&](int r) -> E* {
      return row0 + r < a.R ? x_row<E>(a.o, w.b, w.g, a.G, row0 + r) : nullptr;
    });
  } else {
    const long long ps = ((long long)w.split * a.B * a.Hk + w.bh) * a.R;
    if (ws == 0 && h == 0 && row < a.R) {
      a.part_ml[2 * (ps + row)] = none ? -INFINITY : m;
      a.part_ml[2 * (ps + row) + 1] = none ? 0.f : l;
    }
    x_store<XF32, DP, WR, WS>(acc, mul, none, a.D, threadIdx.x, 0, [&](int r) -> float* {
      return row0 + r < a.R ? a.part + (ps + row0 + r) * a.D : nullptr;
    });
  }
}

// Joins the splits of the forward: one wave per row.
template <class T>
__global__ __launch_bounds__(256) void xattn_fwd_join(const XArgs a) {
  using E = typename T::elem;
  const int lane = threadIdx.x % 64;
  const long long n = (long long)a.B * a.Hk * a.R;
  const long long id = (long long)blockIdx.x * 4 + threadIdx.x / 64;
  if (id >= n) return;
  const int bh = (int)(id / a.R), r = (int)(id % a.R);
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (s * n + id)]);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[4] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * (s * n + id)] - mu);
    l += f * a.part_ml[2 * (s * n + id) + 1];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane + 64 * k < a.D) o[k] += f * a.part[(s * n + id) * a.D + lane + 64 * k];
  }
  const bool none = m == -INFINITY && l == 0.f;
  if (a.lse && lane == 0) a.lse[id] = none ? INFINITY : m + __builtin_amdgcn_logf(l);
  E* p = x_row<E>(a.o, bh / a.Hk, bh % a.Hk, a.G, r);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 64 * k < a.D) p[lane + 64 * k] = T::bits(none ? 0.f : o[k] / l);
}

// ----------------------------------------------------------------- backward ---
// fp16 holds dS from 2^-24 to 2^16 only: dS is scaled by a power of two taken
// from the largest |dO| (of the row for dQ, of all rows for dK, whose sum runs
// over them), and the sum is scaled back in fp32.  bf16 and fp32 need none.
template <class T>
__device__ __forceinline__ float x_down(float amax) {
  if constexpr (std::is_same<T, XF16>::value) {
    const uint32_t e = (__float_as_uint(amax) >> 23) & 255;
    return e == 0 || e == 255 ? 1.f : __uint_as_float((254 - e) << 23);
  }
  return 1.f;
}

// dQ of WR * 32 rows, streaming K and V; also delta (and the rows' |dO|) for
// xattn_dkv, which runs after it.
template <class T, int DP, int WR, int WS, int KT, int OCC>
__global__ __launch_bounds__(64 * WR * WS, OCC) void xattn_dq(const XArgs a) {
  using I = Img<T, DP>;
  using C = FwdCfg<T, DP, WR, WS, KT>;
  using E = typename T::elem;
  const XWork w = x_work(a);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wr = wave % WR, ws = wave / WR;
  const int lr = lane & 31, h = lane >> 5;
  const int rows = x_len(a.q_lens, w.b, a.Tq) * a.G;
  const int row0 = w.tile * WR * 32, row = row0 + wr * 32 + lr;
  const int len = row0 < rows ? x_len(a.kv_lens, w.b, a.Tk) : 0;
  int klo, khi;
  x_share(len, KT, a.splits, w.split, klo, khi);
  const uint8_t* mask = a.mask ? a.mask + w.b * a.mask_sb : nullptr;
  const uint32_t LK = 0, LV = I::bytes(KT);
  const float c2 = a.scale * LOG2E_X;
  const long long at = (long long)w.bh * a.R;

  uint4 qf[I::NC], df[I::NC];
  float delta = 0.f, amax = 0.f;
  {
    const bool live = row < rows;
    const E* p = live ? x_row<E>(a.q, w.b, w.g, a.G, row) : nullptr;
    const E* d = live ? x_row<E>(a.dout, w.b, w.g, a.G, row) : nullptr;
    const E* o = live ? x_row<E>(a.o, w.b, w.g, a.G, row) : nullptr;
#pragma unroll
    for (int j = 0; j < I::NC; ++j) {
      const int ch = 2 * j + h;
      const bool in = live && ch * I::E < a.D;
      qf[j] = in ? ld_chunk<T>(p, ch, a.D) : zero16();
      df[j] = in ? ld_chunk<T>(d, ch, a.D) : zero16();
      const uint4 ov = in ? ld_chunk<T>(o, ch, a.D) : zero16();
      E x[I::E], y[I::E];
      __builtin_memcpy(x, &df[j], 16);
      __builtin_memcpy(y, &ov, 16);
#pragma unroll
      for (int e = 0; e < I::E; ++e) {
        delta = fmaf(T::val(x[e]), T::val(y[e]), delta);
        amax = fmaxf(amax, fabsf(T::val(x[e])));
      }
    }
  }
  delta = xhalf_sum(delta);
  amax = xhalf_max(amax);
  const float L = row < rows ? a.lse[at + row] : INFINITY;
  const float down = x_down<T>(amax);
  if (w.split == 0 && ws == 0 && h == 0 && row < a.R) {
    a.delta[at + row] = delta;
    if (a.amax) a.amax[at + row] = amax;
  }
  f32x16 acc[DP / 32] = {};

  Stage<T, DP, KT, C::NT> sk, sv;
  Keep<KT> kp;
  auto fetch = [&](int k0) {
    kp.load(mask, k0, khi, lane);
    sk.load([&](int r) { return k0 + r < khi ? x_key<E>(a.k, w.b, w.g, k0 + r) : nullptr; }, a.D);
    sv.load([&](int r) { return k0 + r < khi ? x_key<E>(a.v, w.b, w.g, k0 + r) : nullptr; }, a.D);
  };
  if (klo < khi) fetch(klo);
  for (int k0 = klo; k0 < khi; k0 += KT) {
    uint64_t keep[Keep<KT>::W];
    kp.bits(keep);
    __syncthreads();
    sk.store_kept(LK, keep);
    sv.store_kept(LV, keep);
    __syncthreads();
    if (k0 + KT < khi) fetch(k0 + KT);
#pragma unroll
    for (int u = 0; u < C::SUB; ++u) {
      const int r0 = (ws * C::SUB + u) * 32;
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int j = 0; j < I::NC; ++j) {
        s = T::mma(I::rm(LK, r0, j, lane), qf[j], s);
        dp = T::mma(I::rm(LV, r0, j, lane), df[j], dp);
      }
      const uint32_t kb = (uint32_t)(keep[r0 >> 6] >> (r0 & 63));
      if (kb != 0xffffffffu) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = (kb >> acc_row(e, h)) & 1 ? s[e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, -L)) * ((dp[e] - delta) * down);
#pragma unroll
      for (int c = 0; c < I::NPF; ++c) {
        const uint4 p = I::pack(s, c);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] = T::mma(I::tr(LK, r0, c, db, lane), p, acc[db]);
      }
    }
  }
  const float mul = a.scale / down;
  const bool none = L == INFINITY;
  if (a.splits == 1) {
    x_store<T, DP, WR, WS>(acc, mul, none, a.D, threadIdx.x, 0, [&](int r) -> E* {
      return row0 + r < a.R ? x_row<E>(a.dq, w.b, w.g, a.G, row0 + r) : nullptr;
    });
  } else {
    const long long ps = ((long long)w.split * a.B * a.Hk + w.bh) * a.R;
    x_store<XF32, DP, WR, WS>(acc, mul, none, a.D, threadIdx.x, 0, [&](int r) -> float* {
      return row0 + r < a.R ? a.part + (ps + row0 + r) * a.D : nullptr;
    });
  }
}

// dK and dV of WC * 32 states, streaming Q and dO over RT rows at a time; WS
// waves share the states and take different rows, DS waves the columns of the
// results (where both accumulators are too large for one wave's registers).
template <class T, int DP, int WC, int WS, int DS, int RT>
struct DkvCfg {
  static constexpr int NT = 64 * WC * WS * DS;
  static constexpr int SUB = RT / WS / 32;
  static constexpr int ST = 2 * Img<T, DP>::bytes(RT);       // L, delta behind the tiles
  static constexpr int OUT = x_store_bytes<T, DP / DS, WC, WS>();
  static constexpr int OUT32 = x_store_bytes<XF32, DP / DS, WC, WS>();
  static constexpr int LDS = x_max(ST + 8 * RT, DS * OUT);
  static constexpr int LDS32 = x_max(LDS, DS * OUT32);
};

template <class T, int DP, int WC, int WS, int DS, int RT, int OCC>
__global__ __launch_bounds__(64 * WC * WS * DS, OCC) void xattn_dkv(const XArgs a) {
  using I = Img<T, DP>;
  using C = DkvCfg<T, DP, WC, WS, DS, RT>;
  using E = typename T::elem;
  constexpr int DH = DP / DS, NB = DH / 32;
  const XWork w = x_work(a);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int wc = wave % WC, ws = wave / WC % WS, ds = wave / (WC * WS);
  const int lr = lane & 31, h = lane >> 5;
  const int len = x_len(a.kv_lens, w.b, a.Tk);
  const int key0 = w.tile * WC * 32, key = key0 + wc * 32 + lr;
  const int rows = x_len(a.q_lens, w.b, a.Tq) * a.G;
  int rlo, rhi;
  x_share(key0 < len ? rows : 0, RT, a.splits, w.split, rlo, rhi);
  const bool kept = key < len && (!a.mask || a.mask[w.b * a.mask_sb + key]);
  const uint32_t LQ = 0, LD = I::bytes(RT), LL = C::ST, LT = LL + 4 * RT;
  const float c2 = a.scale * LOG2E_X;
  const long long at = (long long)w.bh * a.R;

  float down = 1.f;
  if constexpr (std::is_same<T, XF16>::value) {
    float x = 0.f;
    for (int r = threadIdx.x; r < rows; r += C::NT) x = fmaxf(x, a.amax[at + r]);
    x = wave_max(x);
    if (lane == 0) lds_stf(4 * wave, x);
    __syncthreads();
    for (int i = 0; i < C::NT / 64; ++i) x = fmaxf(x, lds_ldf(4 * i));
    down = x_down<T>(x);
    __syncthreads();
  }

  uint4 kf[I::NC], vf[I::NC];
  {
    const E* p = x_key<E>(a.k, w.b, w.g, kept ? key : 0);
    const E* v = x_key<E>(a.v, w.b, w.g, kept ? key : 0);
#pragma unroll
    for (int j = 0; j < I::NC; ++j) {
      const bool in = kept && (2 * j + h) * I::E < a.D;
      kf[j] = in ? ld_chunk<T>(p, 2 * j + h, a.D) : zero16();
      vf[j] = in ? ld_chunk<T>(v, 2 * j + h, a.D) : zero16();
    }
  }
  f32x16 dk[NB] = {}, dv[NB] = {};

  Stage<T, DP, RT, C::NT> sq, sd;
  float fl = INFINITY, ft = 0.f;
  auto fetch = [&](int r0) {
    sq.load([&](int r) {
      return r0 + r < rhi ? x_row<E>(a.q, w.b, w.g, a.G, r0 + r) : nullptr; }, a.D);
    sd.load([&](int r) {
      return r0 + r < rhi ? x_row<E>(a.dout, w.b, w.g, a.G, r0 + r) : nullptr; }, a.D);
    const int r = r0 + threadIdx.x;
    const bool in = threadIdx.x < RT && r < rhi;
    fl = in ? a.lse[at + r] : INFINITY;
    ft = in ? a.delta[at + r] : 0.f;
  };
  if (rlo < rhi) fetch(rlo);
  for (int t0 = rlo; t0 < rhi; t0 += RT) {
    __syncthreads();
    sq.store(LQ);
    sd.store(LD);
    if (threadIdx.x < RT) {
      lds_stf(LL + 4 * threadIdx.x, fl);
      lds_stf(LT + 4 * threadIdx.x, ft);
    }
    __syncthreads();
    if (t0 + RT < rhi) fetch(t0 + RT);
#pragma unroll
    for (int u = 0; u < C::SUB; ++u) {
      const int r0 = (ws * C::SUB + u) * 32;
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int j = 0; j < I::NC; ++j) {
        s = T::mma(I::rm(LQ, r0, j, lane), kf[j], s);
        dp = T::mma(I::rm(LD, r0, j, lane), vf[j], dp);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 lu = lds_ld16(LL + 4 * (r0 + 8 * k + 4 * h));
        const uint4 tu = lds_ld16(LT + 4 * (r0 + 8 * k + 4 * h));
        const uint32_t *lp = (const uint32_t*)&lu, *tp = (const uint32_t*)&tu;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * k + e;
          s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -__uint_as_float(lp[e])));
          dp[i] = s[i] * ((dp[i] - __uint_as_float(tp[e])) * down);
        }
      }
#pragma unroll
      for (int c = 0; c < I::NPF; ++c) {
        const uint4 p = I::pack(s, c), g = I::pack(dp, c);
#pragma unroll
        for (int db = 0; db < NB; ++db) {
          dv[db] = T::mma(I::tr(LD, r0, c, ds * NB + db, lane), p, dv[db]);
          dk[db] = T::mma(I::tr(LQ, r0, c, ds * NB + db, lane), g, dk[db]);
        }
      }
    }
  }
  const int tid = threadIdx.x % (64 * WC * WS), Dh = min(a.D - ds * DH, DH);
  const float mul = a.scale / down;
  if (a.splits == 1) {
    const auto dst = [&](const XView& v) {
      return [&](int r) -> E* {
        return key0 + r < a.Tk ? x_key<E>(v, w.b, w.g, key0 + r) + ds * DH : nullptr;
      };
    };
    x_store<T, DH, WC, WS>(dk, mul, !kept, Dh, tid, ds * C::OUT, dst(a.dk));
    x_store<T, DH, WC, WS>(dv, 1.f, !kept, Dh, tid, ds * C::OUT, dst(a.dv));
  } else {
    const auto dst = [&](int which) {
      const long long ps =
          (((long long)which * a.splits + w.split) * a.B * a.Hk + w.bh) * a.Tk + key0;
      return [=](int r) -> float* {
        return key0 + r < a.Tk ? a.part + (ps + r) * a.D + ds * DH : nullptr;
      };
    };
    x_store<XF32, DH, WC, WS>(dk, mul, !kept, Dh, tid, ds * C::OUT32, dst(0));
    x_store<XF32, DH, WC, WS>(dv, 1.f, !kept, Dh, tid, ds * C::OUT32, dst(1));
  }
}

// Sums the splits of a gradient, one wave per row: dQ (n rows = R), or dK and
// dV (blockIdx.y, n rows = Tk).
template <class T, bool KV>
__global__ __launch_bounds__(256) void xattn_join(const XArgs a) {
  using E = typename T::elem;
  const int lane = threadIdx.x % 64, per = KV ? a.Tk : a.R;
  const long long n = (long long)a.B * a.Hk * per;
  const long long id = (long long)blockIdx.x * 4 + threadIdx.x / 64;
  if (id >= n) return;
  const int bh = (int)(id / per), r = (int)(id % per), b = bh / a.Hk, g = bh % a.Hk;
  const float* part = a.part + (KV ? blockIdx.y * a.splits * n * a.D : 0);
  E* p = KV ? x_key<E>(blockIdx.y ? a.dv : a.dk, b, g, r) : x_row<E>(a.dq, b, g, a.G, r);
  for (int d = lane; d < a.D; d += 64) {
    float x = 0.f;
    for (int s = 0; s < a.splits; ++s) x += part[(s * n + id) * a.D + d];
    p[d] = T::bits(x);
  }
}

// ------------------------------------------------------------------- launch ---
enum { X_FWD, X_DQ, X_DKV };

struct XPlan {
  int few, tiles, splits;
};
// The split of one kernel's work.  `own` rows (dK, dV: states) belong to the
// waves, 32 each; the others are streamed.  Where 32 (fp32 with 256 columns:
// 64) hold them all, the block's waves share them and take different parts of
// the stream.  Fewer than 512 blocks (two per CU) split the stream further,
// into parts that a second launch joins.
inline XPlan x_plan(const XArgs& a, int type, int what) {
  const int own = what == X_DKV ? a.Tk : a.R, stream = what == X_DKV ? a.R : a.Tk;
  const bool wide = type == 1 && a.D > 128;
  XPlan p;
  p.few = own <= (wide && what != X_DKV ? 64 : 32);
  const int per = wide && what == X_DKV ? 64 : 128;
  p.tiles = p.few ? 1 : (own + per - 1) / per;
  const long long blocks = (long long)p.tiles * a.B * a.Hk;
  const int step = p.few ? 128 : 64, most = (stream + step - 1) / step;
  const long long want = blocks >= 512 ? 1 : (512 + blocks - 1) / blocks;
  p.splits = (int)(want < most ? want : most);
  return p;
}

template <class K>
int x_go(K kernel, const XArgs& a, int lds, int nt, void* stream) {
  if (lds > 64 * 1024)
    if (const int e = set_max_lds((const void*)kernel, lds)) return e;
  const long long grid = (long long)a.tiles * a.splits * a.B * a.Hk;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(nt), lds, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

template <class T, int DP>
int x_run(XArgs a, int what, void* stream) {
  constexpr bool wide = DP * T::ES > 512;               // fp32, 256 columns
  constexpr int OCC = DP * T::ES <= 256 ? 2 : 1;
  constexpr int KT = wide ? 32 : 64;
  constexpr int FR = wide ? 2 : 1, FS = wide ? 2 : 4, FK = wide ? 64 : 128;
  const XPlan p = x_plan(a, T::TYPE, what);
  a.tiles = p.tiles;
  a.splits = p.splits;
  const int nrow = a.B * a.Hk * (what == X_DKV ? a.Tk : a.R);
  int e;
  if (what != X_DKV) {
    using C = FwdCfg<T, DP, 4, 1, KT>;
    using S = FwdCfg<T, DP, FR, FS, FK>;
    constexpr int L = x_max(C::LDS, x_store_bytes<XF32, DP, 4, 1>());
    const int lds = p.few ? S::LDS : a.splits > 1 ? L : C::LDS;
    if (what == X_FWD) {
      e = p.few ? x_go(xattn_fwd<T, DP, FR, FS, FK, 1>, a, lds, S::NT, stream)
                : x_go(xattn_fwd<T, DP, 4, 1, KT, OCC>, a, lds, C::NT, stream);
      if (e || a.splits == 1) return e;
      hipLaunchKernelGGL((xattn_fwd_join<T>), dim3((nrow + 3) / 4), dim3(256), 0,
                         (hipStream_t)stream, a);
      return (int)hipGetLastError();
    }
    e = p.few ? x_go(xattn_dq<T, DP, FR, FS, FK, 1>, a, lds, S::NT, stream)
              : x_go(xattn_dq<T, DP, 4, 1, KT, OCC>, a, lds, C::NT, stream);
    if (e || a.splits == 1) return e;
    hipLaunchKernelGGL((xattn_join<T, false>), dim3((nrow + 3) / 4), dim3(256), 0,
                       (hipStream_t)stream, a);
    return (int)hipGetLastError();
  }
  constexpr int DS = wide ? 2 : 1, RT = 32;
  constexpr int MC = wide ? 2 : 4;                        // states: 32 MC per block
  using C = DkvCfg<T, DP, MC, 1, DS, RT>;
  using S = DkvCfg<T, DP, 1, MC, DS, 32 * MC>;
  e = p.few ? x_go(xattn_dkv<T, DP, 1, MC, DS, 32 * MC, 1>, a, a.splits > 1 ? S::LDS32 : S::LDS,
                   S::NT, stream)
            : x_go(xattn_dkv<T, DP, MC, 1, DS, RT, 1>, a, a.splits > 1 ? C::LDS32 : C::LDS, C::NT,
                   stream);
  if (e || a.splits == 1) return e;
  hipLaunchKernelGGL((xattn_join<T, true>), dim3((nrow + 3) / 4, 2), dim3(256), 0,
                     (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

template <class T>
int x_by_width(const XArgs& a, int what, void* stream) {
  return a.D <= 64 ? x_run<T, 64>(a, what, stream)
                   : a.D <= 128 ? x_run<T, 128>(a, what, stream) : x_run<T, 256>(a, what, stream);
}
int xattn_run_bf16(const XArgs& a, int what, void* stream);
int xattn_run_f16(const XArgs& a, int what, void* stream);
int xattn_run_f32(const XArgs& a, int what, void* stream);

}  // namespace tgfr
