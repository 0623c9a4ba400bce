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
// bf16 / fp16 round P and dS to the type as MFMA operands (2^-8 / 2^-11
// relative, of the size of the one rounding of the result), fp16 scaled by powers
// of two into its range (XF16, DownScale); sums, statistics and accumulators are
// fp32.
//
// Masked states never reach a product: their rows of K and V are written to
// LDS as zeros (NaN or infinity there stays there) and their scores are -inf.
#pragma once
#include <type_traits>

#include "tgfr_common.h"

namespace tgfr {

#define X_INLINE __attribute__((always_inline))
// waves per SIMD, neither fewer nor more: a compiler that hopes for more keeps
// registers free that operands read ahead need
#define X_OCCUPANCY(n) __attribute__((amdgpu_waves_per_eu(n, n)))

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
  float* lse;            // [B Hk][R]: log2 of the row's sum less T::PBITS; +inf: none
  float* delta;          // [B Hk][R]
  float* size;           // [B Hk][R] |dO| of the row (fp16 only)
  float* vmax;           // [B Hk][chunks] squares of the largest |V| (fp16 only)
  float* part;           // partial results of the splits
  float* part_ml;        // forward: [split][B Hk][R][2] maximum and sum
  int B, Tq, Tk, H, Hk, G, D, R;   // R = Tq G
  int splits, tiles, chunks;
  int fast_k, fast_q;              // rows may be read as whole aligned chunks, tile by tile
  uint32_t per_g;                  // 2^32 / G, rounded up; 0 for G = 1
  float scale;
};

struct XBf16 {
  static constexpr int TYPE = 0, ES = 2, PBITS = 0, LAG = 8, UP = 0;
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
  // The backward's probabilities are held times 2^14: fp16 has all its digits from
  // 2^-14 on only, and even attention to 2^19 states gives each 2^-19.
  static constexpr int PBITS = 14;
  // The forward's, relative to the running maximum, stay below 2^(LAG + UP) and
  // begin to lose digits at 2^(-14 - UP): many states far below one count.
  static constexpr int LAG = 4, UP = 11;
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
  static constexpr int TYPE = 1, ES = 4, PBITS = 0, LAG = 8, UP = 0;
  static constexpr bool VEC = true;       // rows of whole 16-byte chunks
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

struct XF32Any : XF32 {
  static constexpr bool VEC = false;
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
  // B operand c (r0 a multiple of 32); 16-bit types
  static __device__ __forceinline__ uint4 tr(uint32_t base, int r0, int c, int db, int lane) {
    const int i = lane & 15, g = lane >> 4, h = g >> 1, q = i >> 2;
    const int ch = 4 * db + 2 * (g & 1) + ((i >> 1) & 1), in = 8 * (i & 1);
    s16x4 v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * e + 4 * h + q;            // + 16 c + r0: f is the same
      v[e] = lds_tr4(base + (r0 + 16 * c) * ROWB + r * ROWB + ((ch ^ f(r)) << 4) + in);
    }
    return __builtin_bit_cast(uint4, join_tr(v[0], v[1]));
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

// A buffer over a tile: its rows lie within 2^31 bytes of its first (the entries
// check the strides), and a lane offset of NONE reads zeros.
constexpr uint32_t NONE = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* p) {
  return uniform_rsrc(p, NONE);
}
__device__ __forceinline__ uint4 buf16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ __forceinline__ uint32_t buf4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
}

// zeros for places that are not read, then the statistics of such rows (log
// sum +infinity: probability 0; delta 0)
static __device__ const float x_pad[8] __attribute__((aligned(16))) = {
    0.f, 0.f, 0.f, 0.f, INFINITY, 0.f, 0.f, 0.f};
__device__ __forceinline__ const void* scalar(const void* p) {
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)p);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)p >> 32));
  return (const void*)(lo | (hi << 32));
}
// 16 bytes per lane of `lanes` from a scalar base + lane offset (4 of every lane
// from an address) straight to LDS byte `to` (wave-uniform) + 16 (4) * lane.
// Inline asm, so that the compiler sees no LDS write pending on the memory
// counter; the kernels wait by count (glds16).  Lanes are chosen by exec, not by
// branches: around those the accumulators were moved from register to register
// (dK and dV of 4 x 1024 rows, 16 heads of 128 on 4, on 1500 states: 149 us
// against 161).  The s_nop completes the five wait states that a scalar register
// written by a vector instruction (readfirstlane: the base) needs before a
// memory instruction reads it, which the compiler cannot see to in here.
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t to,
                                      uint64_t lanes) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_base() + to));
  uint64_t all;
  asm volatile("s_mov_b64 %0, exec\n\ts_mov_b32 m0, %3\n\ts_and_b64 exec, exec, %4\n\t"
               "s_nop 1\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, %0"
               : "=&s"(all)
               : "v"(off), "s"(scalar(base)), "s"(m0), "s"(lanes)
               : "memory", "m0", "scc");
}
__device__ __forceinline__ void dma4(const float* src, uint32_t to) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_base() + to));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(m0)
               : "memory", "m0");
}

// Feeds tiles of ROWS rows (16-bit types) to LDS images by DMA, which takes no
// registers: a wave's instruction fills 1 KiB of the image in lane order, so
// the lanes fetch the chunks that the image's swizzle puts there.  A thread's
// chunks lie at fixed offsets from the tile's first row: a whole tile costs no
// address arithmetic but the scalar base's.
template <class T, int DP, int ROWS, int NT>
struct Feed {
  using I = Img<T, DP>;
  static constexpr int N = ROWS * I::CPR / NT;
  static_assert(ROWS * I::CPR % NT == 0, "whole instructions");
  uint32_t off[N], wave;     // (the wave's first place)
  uint64_t lanes[N];         // whose chunks are part of a row

  static __device__ __forceinline__ int row(int n) { return (threadIdx.x + NT * n) / I::CPR; }
  static __device__ __forceinline__ int chunk(int n) {
    return (int)(threadIdx.x + NT * n) % I::CPR ^ I::f(row(n));
  }
  static __device__ __forceinline__ uint32_t place(int n) { return 16 * (threadIdx.x + NT * n); }

  // at(i): byte offset of row i from the tile's first
  template <class At>
  __device__ __forceinline__ void init(At at, int D) {
    wave = __builtin_amdgcn_readfirstlane(16 * (threadIdx.x & ~63u));
#pragma unroll
    for (int n = 0; n < N; ++n) {
      off[n] = chunk(n) * I::E < D ? at(row(n)) + 16 * chunk(n) : NONE;
      lanes[n] = __ballot(off[n] != NONE);
    }
  }
  // columns past D, once: the feed leaves them alone
  __device__ __forceinline__ void clear(uint32_t base) const {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (off[n] == NONE) lds_st16(base + place(n), zero16());
  }
  // starts a whole tile whose first row is at p; N DMA instructions per wave (an
  // instruction covers whole rows: some lanes always take part)
  __device__ __forceinline__ void start(const void* p, uint32_t base) const {
#pragma unroll
    for (int n = 0; n < N; ++n) dma16(p, off[n], base + wave + 16 * NT * n, lanes[n]);
  }
  // the same with zeros for the rows that are not kept(row), which are not
  // read: their lanes fetch zeros from x_pad
  template <class Kept>
  __device__ __forceinline__ void start_kept(const void* p, Kept kept, uint32_t base) const {
#pragma unroll
    for (int n = 0; n < N; ++n)
      glds16(off[n] != NONE && kept(row(n)) ? (const char*)p + off[n] : (const char*)x_pad,
             base + wave + 16 * NT * n);
  }
  // the same for rows at any alignment and of any length, through registers:
  // at(i) points to row i of the tile, or is NULL for zeros.  No tile is fed
  // beside another's work here (16 heads of 128 on 4, 4 x 1024 x 1500, forward /
  // backward: rows at 2 bytes 114 / 724 us, at 4 bytes or more 60 / 236; 100
  // columns 132 / 827, 104 columns 57 / 230; 12 heads on 4, whose groups of 3
  // straddle tiles in dK and dV alone, 50 / 452, on 6 50 / 208)
  template <class Row>
  __device__ __forceinline__ void copy(Row at, int D, uint32_t base) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const typename T::elem* p = at(row(n));
      lds_st16(base + place(n), p && chunk(n) * I::E < D ? ld_chunk<T>(p, chunk(n), D) : zero16());
    }
  }
};

// Where a kernel's A operands of 32 streamed rows come from.  16-bit types:
// from their tile in LDS.
template <class T, int DP>
struct LdsSrc {
  using I = Img<T, DP>;
  uint32_t base;
  int lane;
  __device__ __forceinline__ uint4 rm(int j) const { return I::rm(base, 0, j, lane); }
  __device__ __forceinline__ uint4 tr(int c, int db) const {
    return I::tr(base, 0, c, db, lane);
  }
};
// fp32: straight from global memory.  Its matrix instructions take 8 times as
// long per byte as bf16's, so cache reads hide behind them without a tile in
// LDS; what counts is loads in flight, so a wave takes 64 columns (below).
template <int DP, bool VEC, class At>
struct MemSrc {
  __amdgpu_buffer_rsrc_t b;
  At at;
  uint32_t row, live, tro[16];
  int lane, D;
  // the 32 rows whose first is at p (D: elements from there on); at(i): byte
  // offset of row i; bit i of `live`: row i exists (others are zeros)
  __device__ __forceinline__ MemSrc(const void* p, At at_, uint32_t live_, int lane_, int D_)
      : b(tile_rsrc(p)), at(at_), live(live_), lane(lane_), D(D_) {
    const int r = lane & 31;
    row = at(r) | (~live >> r) << 31;
    // opaque: offsets formed from it at each use, not kept over the loop
    asm volatile("" : "+v"(row));
  }
  __device__ __forceinline__ uint4 rm(int j) const {
    const int d0 = 8 * j + 4 * (lane >> 5);
    if constexpr (VEC) return buf16(b, d0 < D ? row + 4 * d0 : NONE);
    return make_uint4(buf4(b, d0 < D ? row + 4 * d0 : NONE),
                      buf4(b, d0 + 1 < D ? row + 4 * d0 + 4 : NONE),
                      buf4(b, d0 + 2 < D ? row + 4 * d0 + 8 : NONE),
                      buf4(b, d0 + 3 < D ? row + 4 * d0 + 12 : NONE));
  }
  // before the first tr(): the rows' offsets, kept no longer than needed
  __device__ __forceinline__ void open() {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int q = acc_row(i, lane >> 5);
      tro[i] = (at(q) + 4 * (lane & 31)) | (~live >> q) << 31;     // no branch; at() < NONE
    }
  }
  __device__ __forceinline__ uint4 tr(int c, int db) const {
    const bool in = 32 * db + (lane & 31) < D;
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = buf4(b, in ? tro[4 * c + e] + 128 * db : NONE);
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
};
// the same with all transposed operands read at once, before they are needed
template <int DP, bool VEC, class At>
struct HeldSrc : MemSrc<DP, VEC, At> {
  using Src = MemSrc<DP, VEC, At>;
  uint4 f[4 * (DP / 32)];
  template <class... A>
  __device__ __forceinline__ HeldSrc(A... a) : Src(a...) {
    Src::open();
#pragma unroll
    for (int i = 0; i < 4 * (DP / 32); ++i)
      f[i] = Src::tr(i / (DP / 32), i % (DP / 32));
  }
  __device__ __forceinline__ const uint4& tr(int c, int db) const { return f[c * (DP / 32) + db]; }
};

// ------------------------------------------------------------ shared parts ---
// The block's work: sample, key head, tile of rows (or states), split.
struct XWork {
  int b, g, bh, tile, split;
};
// Place L of `total` along the blocks: consecutive places share K and V (or Q
// and dO), and so should share one XCD's L2.  Where streams differ in length,
// whole samples per XCD would leave the XCDs of short ones idle: runs of four
// (4 x 1024 rows, 16 heads of 128 on 4, on 375 to 1500 states: forward 44 us
// against 58, backward 174 against 183; one token each of 16 samples: 90 both ways).
__device__ __forceinline__ int x_place(int L, int total, bool ragged) {
  if (!ragged) return xcd_remap(L, total);
  const int q = L / 8;
  return L < total / 32 * 32 ? (q / 4 * 8 + L % 8) * 4 + q % 4 : L;
}
// own, stream: lengths (or NULL) of what the waves own, of `per` items per tile
// (tokens of Q count G rows), and of what they stream.
__device__ __forceinline__ XWork x_work(const XArgs& a, const int* own, int T, int G, int per,
                                        const int* stream) {
  XWork w;
  const int L = blockIdx.x, heads = a.Hk * a.splits;
  // Compacting reads all samples' lengths in every block, so its cost grows with
  // the square of the batch: 4096 samples of 20 tokens on 62 states, 4 heads of 64,
  // forward 866 us against 171, 64 of them 7.2 against 6.7 (one tile each: nothing
  // to compact); 512 of 196 on 200, 4 heads of 128 on 2, backward 330 against 371.
  if (!own || a.tiles == 1 || a.B > 512) {
    const int id = x_place(L, gridDim.x, stream);
    w.tile = id % a.tiles;
    const int rest = id / a.tiles;
    w.bh = rest % (a.B * a.Hk);
    w.split = rest / (a.B * a.Hk);
  } else {
    // Tiles of padding only clear their results: they come last, so that the
    // others spread evenly over the CUs.  Lane i counts sample b0 + i's tiles.
    const int lane = threadIdx.x % 64;
    auto tiles_of = [&](int b) {
      return b < a.B ? (min(max(own[b], 0), T) * G + per - 1) / per : 0;
    };
    int live = 0;
    for (int b = lane; b < a.B; b += 64) live += tiles_of(b);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) live += __shfl_xor(live, m);
    live *= heads;
    const bool pad = L >= live;
    const int id = pad ? L - live : x_place(L, live, stream);
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int b = b0 + lane, used = tiles_of(b);
      const int n = b < a.B ? (pad ? a.tiles - used : used) : 0;
      int sum = n;                                       // of the samples up to b
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int up = __shfl_up(sum, m);
        if (lane >= m) sum += up;
      }
      const int lo = (before + sum - n) * heads;
      const uint64_t at = __ballot(id >= lo && id < lo + n * heads);
      if (at) {
        const int k = __builtin_ctzll(at);
        const int r = id - __shfl(lo, k), nk = __shfl(n, k), rest = r / nk;
        w.tile = r % nk + (pad ? __shfl(used, k) : 0);
        w.bh = (b0 + k) * a.Hk + rest % a.Hk;
        w.split = rest / a.Hk;
        break;
      }
      before += __shfl(sum, 63);
    }
  }
  w.b = w.bh / a.Hk;
  w.g = w.bh % a.Hk;
  // (division runs on the vector unit; these are the same in all lanes)
  for (int* p : {&w.tile, &w.bh, &w.split, &w.b, &w.g}) *p = __builtin_amdgcn_readfirstlane(*p);
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
  lo = __builtin_amdgcn_readfirstlane(min(n, split * per * tile));
  hi = __builtin_amdgcn_readfirstlane(min(n, (split + 1) * per * tile));
}
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

// ------------------------------------------------------------ the key stream ---
// The states of a split, a tile of KT = 32 WS at a time, as the forward and dQ
// read them: WR waves along the rows (32 each) x WS waves along the states of
// a tile (a piece of 32 each) x DS waves along the columns.
//
// fp32 with more than 64 columns: DS waves take 64 columns each of Q, K, V and
// the result.  Each forms its part of the scores, the parts are exchanged
// through LDS and summed by all in one order, so a wave's operands and
// accumulators are a quarter of 256 columns' and its loads stay in flight.
// One step in the order in which it is to run: RM products of the scores (of
// the piece ahead), whose operands rm(i) are read AHEAD products early and
// beside which beside(i) runs (the vector work of the current piece, after
// early() has read what it needs), then TR products with operands tr(i).  KEEP
// holds the compiler to this order, which else reads operands two at a time
// right before their products.  Alone on its SIMD a wave of dK, dV needs that
// (167 -> 161 us at 4 x 1024 rows, 16 heads of 128 on 4, on 1500 states; 212 ->
// 177 us at 4 x 1024 x 1024, 8 heads of 256 on 2), and dQ of up to 128 columns
// gains a little (34 -> 33 us at 3 x 333 x 777, 6 heads of 80 on 3); the
// forward (31 -> 32) and dQ of 256 columns (85 -> 88) do not, and where two waves
// share a SIMD it costs registers that they lack.
template <int RM, int TR, int AHEAD, bool KEEP, class Rm, class Mma1, class Early, class Beside,
          class Between, class Tr, class Mma2>
__device__ __forceinline__ void x_step(Rm rm, Mma1 mma1, Early early, Beside beside,
                                       Between between, Tr tr, Mma2 mma2) {
  uint4 f[AHEAD];
  auto load = [&](int i) X_INLINE { return i < RM ? rm(i) : tr(i - RM); };
  auto keep = []() X_INLINE {
    if constexpr (KEEP) __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (i < RM + TR) f[i] = load(i);
  keep();
  early();
  keep();
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    mma1(i, f[i % AHEAD]);
    if (i + AHEAD < RM + TR) f[i % AHEAD] = load(i + AHEAD);
    beside(i);
    keep();
  }
  between();
  keep();
#pragma unroll
  for (int i = RM; i < RM + TR; ++i) {
    mma2(i - RM, f[i % AHEAD]);
    if (i + AHEAD < RM + TR) f[i % AHEAD] = load(i + AHEAD);
    keep();
  }
}
struct XNone {
  template <class... A>
  __device__ __forceinline__ void operator()(A&&...) const {}
};
struct XNoOperand {
  __device__ __forceinline__ uint4 operator()(int) const { return uint4{}; }
};

// The ring of four slots in LDS that 16-bit kernels stream through: piece n
// lies in slot n % 4.  Step n forms the scores of piece n + 1 beside the rest
// of piece n, so that matrix and vector instructions of one wave have
// independent work to overlap; pieces n + 2 and n + 3 are being fed meanwhile.
//   wait(n): piece n + 1 has arrived, all waves are past step n - 1; feeds n + 3
//   first(sp, slot): scores of the piece there;  before(sp, n): what branches
//   on them;  step(sp, slot, next, slot): the rest of a piece and the scores
//   of the next;  last(sp, slot): the rest
// PLAIN steps (whole tiles, nothing masked: `plain` of them) come four at a
// time with constant slots, so that LDS addresses cost nothing.
template <int N, class Wait, class First, class Before, class Step, class Last>
__device__ __forceinline__ void x_pipe(int np, int plain, Wait wait, First first, Before before,
                                       Step step, Last last) {
  using Any = std::false_type;
  using Plain = std::true_type;
  if (np <= 0) return;
  f32x16 now[N], next[N];
  wait(-1, Any{});
  first(now, 0);
  int n = 0;
  for (; n + 4 <= plain; n += 4) {
    wait(n, Plain{});
    before(now, n, Plain{});
    step(now, 0, next, 1);
    wait(n + 1, Plain{});
    before(next, n + 1, Plain{});
    step(next, 1, now, 2);
    wait(n + 2, Plain{});
    before(now, n + 2, Plain{});
    step(now, 2, next, 3);
    wait(n + 3, Plain{});
    before(next, n + 3, Plain{});
    step(next, 3, now, 0);
  }
  for (; n + 1 < np; ++n) {
    wait(n, Any{});
    before(now, n, Any{});
    step(now, n & 3, next, (n + 1) & 3);
#pragma unroll
    for (int i = 0; i < N; ++i) now[i] = next[i];
  }
  wait(n, Any{});
  before(now, n, Any{});
  last(now, n & 3);
}

// Kept bits of up to MAX states in LDS, one word per 32: a mask is read once,
// before the ring, so that no load of it waits behind a feed.
struct XBits {
  static constexpr int MAX = 32768, BYTES = MAX / 8;
};

template <class T, int DP, int WR, int WS, int DS, bool FWD>
struct KeyStream {
  using I = Img<T, DP>;
  using E = typename T::elem;
  static constexpr int NT = 64 * WR * WS * DS, KT = 32 * WS, DH = DP / DS;
  static constexpr bool MEM = T::ES == 4;
  // operands read ahead: as many as the registers hold
  static constexpr int N = FWD ? 1 : 2, AHEAD = MEM ? 8 : FWD || DP == 64 ? 4 : 2;
  static constexpr int TILE = MEM ? 0 : I::bytes(KT), SLOT = 2 * TILE;
  // the ring and the mask's bits (fp32: two exchanges of 8 KiB per wave);
  // later the result
  static constexpr int BITS = 4 * SLOT;
  static constexpr int FED = MEM ? (DS > 1 ? 2 * 8192 * WR * WS * DS : 0) : BITS + XBits::BYTES;
  static constexpr int STAT = 2 * 4 * 32 * WR * WS;
  static constexpr int OUT = x_store_bytes<T, DH, WR, WS>();
  static constexpr int OUT32 = x_store_bytes<XF32, DH, WR, WS>();
  static constexpr int LDS = x_max(x_max(FED, DS * OUT), STAT);
  static constexpr int LDS32 = x_max(x_max(FED, DS * OUT32), STAT);

  // before(sp, kept bits) and work(first, rest, sp, K, V, next, next K, next V)
  // for the pieces of 32 states: sources of their operands; first, rest: which
  // parts of a step to do (true_type).  All waves of the block take part.
  template <class Before, class Work>
  static __device__ __forceinline__ void run(const XArgs& a, const XWork& w, int klo, int khi,
                                             int ws, int ds, Before before, Work work) {
    using Yes = std::true_type;
    using No = std::false_type;
    const int lane = threadIdx.x % 64;
    const uint8_t* mask = a.mask ? a.mask + w.b * a.mask_sb : nullptr;
    const E* K = x_key<E>(a.k, w.b, w.g, 0) + ds * DH;
    const E* V = x_key<E>(a.v, w.b, w.g, 0) + ds * DH;
    const uint32_t kst = (uint32_t)a.k.st * T::ES, vst = (uint32_t)a.v.st * T::ES;
    if constexpr (MEM) {
      for (int t0 = klo; t0 < khi; t0 += KT) {
        const int k0 = t0 + 32 * ws, j = k0 + (lane & 31);
        const uint32_t kb = (uint32_t)__ballot(j < khi && (!mask || mask[j]));
        if (DS == 1 && !kb) continue;
        auto at_k = [=](int r) X_INLINE { return r * kst; };
        auto at_v = [=](int r) X_INLINE { return r * vst; };
        using K_ = decltype(at_k);
        using V_ = decltype(at_v);
        const int Dh = a.D - ds * DH;
        // the second product's operands (of V; dQ: of K) are read at the start
        const std::conditional_t<FWD, MemSrc<DH, T::VEC, K_>, HeldSrc<DH, T::VEC, K_>> ks(
            K + k0 * a.k.st, at_k, kb, lane, Dh);
        const std::conditional_t<FWD, HeldSrc<DH, T::VEC, V_>, MemSrc<DH, T::VEC, V_>> vs(
            V + k0 * a.v.st, at_v, kb, lane, Dh);
        f32x16 sp[N];
        work(Yes{}, No{}, sp, ks, vs, sp, ks, vs);
        before(sp, kb);
        work(No{}, Yes{}, sp, ks, vs, sp, ks, vs);
      }
    } else {
      static_assert(DS == 1, "whole rows");
      for (int c = klo; c < khi; c += XBits::MAX)
        part(a, mask, K, V, kst, vst, c, min(khi, c + XBits::MAX), ws, before, work);
    }
  }

  template <class Before, class Work>
  static __device__ __forceinline__ void part(const XArgs& a, const uint8_t* mask, const E* K,
                                              const E* V, uint32_t kst, uint32_t vst, int klo,
                                              int khi, int ws, Before before, Work work) {
    using Yes = std::true_type;
    using No = std::false_type;
    const int lane = threadIdx.x % 64;
    using F = Feed<T, DP, KT, NT>;
    F fk, fv;
    fk.init([&](int r) { return r * kst; }, a.D);
    fv.init([&](int r) { return r * vst; }, a.D);
    __syncthreads();                         // the LDS may have been in use
    for (int i = 0; i < 4; ++i) {
      fk.clear(i * SLOT);
      fv.clear(i * SLOT + TILE);
    }
    const int np = (khi - klo + KT - 1) / KT, full = (khi - klo) / KT;
    // kept bits of 32 states from klo + 32 i on (any i), the same in all lanes
    auto bits = [&](int i) X_INLINE -> uint32_t {
      const int left = khi - klo - 32 * i;
      if (left <= 0) return 0;
      if (mask)
        return __builtin_amdgcn_readfirstlane(
            *(LDS_AS uint32_t*)(lds_base() + BITS + 4 * i));
      return left >= 32 ? 0xffffffffu : (1u << left) - 1;
    };
    auto feed = [&](int n) X_INLINE {
      const int k0 = klo + n * KT;
      const uint32_t l0 = (n & 3) * SLOT;
      if (n >= np) return;
      if (a.fast_k && !mask && n < full) {
        fk.start(K + k0 * a.k.st, l0);
        fv.start(V + k0 * a.v.st, l0 + TILE);
        return;
      }
      uint32_t kb[WS];
#pragma unroll
      for (int i = 0; i < WS; ++i) kb[i] = bits(n * WS + i);
      auto kept = [&](int r) X_INLINE {
        uint32_t word = kb[0];
#pragma unroll
        for (int i = 1; i < WS; ++i) word = r >> 5 == i ? kb[i] : word;
        return (word >> (r & 31)) & 1;
      };
      if (a.fast_k) {
        fk.start_kept(K + k0 * a.k.st, kept, l0);
        fv.start_kept(V + k0 * a.v.st, kept, l0 + TILE);
      } else {
        fk.copy([&](int r) X_INLINE { return kept(r) ? K + (k0 + r) * a.k.st : nullptr; }, a.D, l0);
        fv.copy([&](int r) X_INLINE { return kept(r) ? V + (k0 + r) * a.v.st : nullptr; }, a.D, l0 + TILE);
      }
    };
    if (mask) {
      for (int j = klo + (threadIdx.x & ~63); j < khi; j += NT) {
        const uint64_t b = __ballot(j + lane < khi && mask[j + lane]);
        if (lane < 2)
          *(LDS_AS uint32_t*)(lds_base() + BITS + 4 * ((j - klo) / 32 + lane)) = b >> (32 * lane);
      }
      __syncthreads();
    }
    feed(0);
    feed(1);
    feed(2);
    auto wait = [&](int n, auto plain) X_INLINE {
      if constexpr (plain.value) {
        ring_barrier<2 * F::N>();            // all but piece n + 2
        const int k0 = klo + (n + 3) * KT;
        const uint32_t l0 = ((n + 3) & 3) * SLOT;
        fk.start(K + k0 * a.k.st, l0);
        fv.start(V + k0 * a.v.st, l0 + TILE);
      } else {
        if (a.fast_k && n >= 0 && n + 2 < np)
          ring_barrier<2 * F::N>();
        else
          ring_barrier<0>();
        if (n >= 0) feed(n + 3);
      }
    };
    const uint32_t mine = I::bytes(32) * ws;
    auto src = [&](uint32_t at) { return LdsSrc<T, DP>{at + mine, lane}; };
    auto K_ = [&](int slot) X_INLINE { return src(slot * SLOT); };
    auto V_ = [&](int slot) X_INLINE { return src(slot * SLOT + TILE); };
    x_pipe<N>(
        np, a.fast_k && !mask ? full - 3 : 0, wait,
        [&](f32x16 (&sp)[N], int s) X_INLINE {
          work(Yes{}, No{}, sp, K_(s), V_(s), sp, K_(s), V_(s));
        },
        [&](f32x16 (&sp)[N], int n, auto plain) X_INLINE {
          before(sp, plain.value ? 0xffffffffu : bits(n * WS + ws));
        },
        [&](f32x16 (&sp)[N], int s, f32x16 (&next)[N], int t) X_INLINE {
          work(Yes{}, Yes{}, sp, K_(s), V_(s), next, K_(t), V_(t));
        },
        [&](f32x16 (&sp)[N], int s) X_INLINE {
          work(No{}, Yes{}, sp, K_(s), V_(s), sp, K_(s), V_(s));
        });
  }
};

// Sums a score tile over the DS waves that formed parts of it (N tiles per
// exchange); `turn` alternates between two places, so one barrier is enough.
template <int DS, int N>
__device__ __forceinline__ void x_exchange(f32x16 (&s)[N], int group, int ds, int& turn) {
  if constexpr (DS > 1) {
    const int lane = threadIdx.x % 64;
    const uint32_t base = (turn * (int)(blockDim.x / 64) + group * DS) * 8192 + 16 * lane;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        lds_st16(base + ds * 8192 + 4096 * n + 1024 * k,
                 make_uint4(__float_as_uint(s[n][4 * k]), __float_as_uint(s[n][4 * k + 1]),
                            __float_as_uint(s[n][4 * k + 2]), __float_as_uint(s[n][4 * k + 3])));
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x4 v = __builtin_bit_cast(f32x4, lds_ld16(base + 4096 * n + 1024 * k));
#pragma unroll
        for (int x = 1; x < DS; ++x)
          v += __builtin_bit_cast(f32x4, lds_ld16(base + x * 8192 + 4096 * n + 1024 * k));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][4 * k + e] = v[e];
        __builtin_amdgcn_sched_barrier(0);       // or all parts are in registers at once
      }
    turn ^= 1;
  }
}

// B operands of 32 rows, one per lane, held in registers.
template <class T, int DP>
struct Rows32 {
  using I = Img<T, DP>;
  uint4 f[I::NC];
  // p: the lane's row, or NULL for zeros, of D elements
  __device__ __forceinline__ void load(const typename T::elem* p, int D, int h) {
    bool chunks = D % I::E == 0;
    if constexpr (T::ES == 4) chunks = T::VEC;
    if (chunks) {                  // no branches, so all loads are in flight together
#pragma unroll
      for (int j = 0; j < I::NC; ++j) {
        const int d = (2 * j + h) * I::E;
        f[j] = __builtin_bit_cast(
            uint4, (u32x4) * (const u32x4_u*)(p && d < D ? (const void*)(p + d) : x_pad));
      }
    } else {
#pragma unroll
      for (int j = 0; j < I::NC; ++j)
        f[j] = p && (2 * j + h) * I::E < D ? ld_chunk<T>(p, 2 * j + h, D) : zero16();
    }
  }
  __device__ __forceinline__ const uint4& operator[](int j) const { return f[j]; }
};

// scores of masked states
__device__ __forceinline__ void x_mask(f32x16& s, uint32_t kb, int h) {
  if (kb != 0xffffffffu) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = (kb >> acc_row(e, h)) & 1 ? s[e] : -INFINITY;
  }
}

// A row's statistic for the backward.  Past 2^22, where fp32's steps make exponents
// inexact by 2^-2 and more, fp16 takes it a step high: P stays in the type.
template <class T>
__device__ __forceinline__ float x_lse(float m, float l) {
  const float x = m + __builtin_amdgcn_logf(l) - T::PBITS;
  return T::PBITS && fabsf(x) >= 0x1p22f ? fmaf(fabsf(x), 0x1p-23f, x) : x;
}

// ------------------------------------------------------------------ forward ---
// 4 x 2048 rows of 16 heads of 128 on 4 x 4096 states of 4, bf16: 261 us, 1050
// TFLOP/s, bound by the matrix units (a library product of 8192^3: 1172).  One
// token, 16 samples, 32 heads on 8, up to 8192 states: 72 us, 4.8 TB/s, bound by
// reading K and V.  fp32, 64 x 30 rows on 196 states of 256: 15 us, bound by the
// latency of its 4 splits' two pieces; 4 x 1024 rows of 16 heads of 128 on 4 x 1500
// states of 4: 473 us, 106 TFLOP/s of 153; one token, 16 samples, 32 heads on 8, 8192
// states: 226 us, 4.7 TB/s.
template <class T, int DP, int WR, int WS, int DS, int OCC>
__global__ __launch_bounds__(64 * WR * WS * DS) X_OCCUPANCY(OCC) void xattn_fwd(const XArgs a) {
  using S = KeyStream<T, DP, WR, WS, DS, true>;
  using I = Img<T, S::DH>;
  using E = typename T::elem;
  const XWork w = x_work(a, a.q_lens, a.Tq, a.G, 32 * WR, a.kv_lens);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int wr = wave % WR, ws = wave / WR % WS, ds = wave / (WR * WS);
  const int lr = lane & 31, h = lane >> 5;
  const int rows = x_len(a.q_lens, w.b, a.Tq) * a.G;
  const int row0 = w.tile * WR * 32, row = row0 + wr * 32 + lr;
  const int len = row0 < rows ? x_len(a.kv_lens, w.b, a.Tk) : 0;
  int klo, khi;
  x_share(len, S::KT, a.splits, w.split, klo, khi);
  const float c2 = a.scale * LOG2E_X;

  const int Dh = a.D - ds * S::DH;           // columns from this wave's first on
  Rows32<T, S::DH> qf;
  qf.load(row < rows ? x_row<E>(a.q, w.b, w.g, a.G, row) + ds * S::DH : nullptr, Dh, h);
  constexpr int NB = S::DH / 32;
  f32x16 acc[NB] = {};
  int turn = 0;
  // the reference that exponents are taken against, in the log2 domain:
  // exp(scale s - max) = 2^(c2 s - m).  It follows the running maximum only
  // once that has grown by LAG: sums and accumulators, relative to it, stay
  // exact, probabilities stay below 2^(LAG + UP), and most tiles rescale nothing.
  // (Past 2^22 the fp32 steps of m would take the place of UP: it is left out.)
  auto reference = [&](float top) X_INLINE {
    return T::UP && fabsf(top) < 0x1p22f ? top - T::UP : top;
  };
  float m = -INFINITY, l = 0.f;

  auto before = [&](f32x16 (&sp)[1], uint32_t kb) X_INLINE {
    f32x16& s = sp[0];
    x_mask(s, kb, h);
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
    top = reference(xhalf_max(top) * c2);
    if (__any(top > m + T::LAG || m == -INFINITY)) {
      const float mn = fmaxf(m, top);
      const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int db = 0; db < S::DH / 32; ++db) acc[db] *= al;
    }
  };
  S::run(a, w, klo, khi, ws, ds, before,
         [&](auto first, auto rest, f32x16 (&sp)[1], const auto&, const auto& vs,
             f32x16 (&next)[1], const auto& kn, const auto&) X_INLINE {
    constexpr bool A = first.value, B = rest.value;
    constexpr int RM = A ? I::NC : 0, TR = B ? I::NPF * NB : 0, PER = 16 / I::NC;
    const float mu = m == -INFINITY ? 0.f : m;        // no kept state so far
    uint4 p[I::NPF];
    auto probability = [&](int e) X_INLINE {
      sp[0][e] = __builtin_amdgcn_exp2f(fmaf(sp[0][e], c2, -mu));
      l += sp[0][e];
    };
    if constexpr (A) next[0] = f32x16{};
    x_step<RM, TR, S::AHEAD, false>(
        [&](int i) X_INLINE { return kn.rm(i); },
        [&](int i, uint4 f) X_INLINE { next[0] = T::mma(f, qf[i], next[0]); },
        []() X_INLINE {},
        [&](int i) X_INLINE {
          if constexpr (B)
#pragma unroll
            for (int e = i * PER; e < (i + 1) * PER; ++e) probability(e);
        },
        [&]() X_INLINE {
          if constexpr (B) {
            if constexpr (!A)
#pragma unroll
              for (int e = 0; e < 16; ++e) probability(e);
#pragma unroll
            for (int c = 0; c < I::NPF; ++c) p[c] = I::pack(sp[0], c);
          }
        },
        [&](int i) X_INLINE { return vs.tr(i / NB, i % NB); },
        [&](int i, uint4 f) X_INLINE { acc[i % NB] = T::mma(f, p[i / NB], acc[i % NB]); });
    if constexpr (A && !B) x_exchange<DS>(next, ws * WR + wr, ds, turn);
  });
  l = xhalf_sum(l);

  float mul = 1.f;
  if constexpr (WS > 1) {       // the waves that share rows agree on the reference
    constexpr uint32_t ML = 0;
    __syncthreads();
    if (h == 0 && ds == 0) {
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
  const bool none = !(row < rows) || (m == -INFINITY && l == 0.f);
  const int tid = threadIdx.x % (64 * WR * WS);
  const long long at = (long long)w.bh * a.R;
  if (a.splits == 1) {
    if (a.lse && ws == 0 && ds == 0 && h == 0 && row < a.R)
      a.lse[at + row] = none ? INFINITY : x_lse<T>(m, l);
    x_store<T, S::DH, WR, WS>(acc, mul / l, none, Dh, tid, ds * S::OUT, [&](int r) -> E* {
      return row0 + r < a.R ? x_row<E>(a.o, w.b, w.g, a.G, row0 + r) + ds * S::DH : nullptr;
    });
  } else {
    const long long ps = ((long long)w.split * a.B * a.Hk + w.bh) * a.R;
    if (ws == 0 && ds == 0 && h == 0 && row < a.R) {
      a.part_ml[2 * (ps + row)] = none ? -INFINITY : m;
      a.part_ml[2 * (ps + row) + 1] = none ? 0.f : l;
    }
    x_store<XF32, S::DH, WR, WS>(acc, mul, none, Dh, tid, ds * S::OUT32, [&](int r) -> float* {
      return row0 + r < a.R ? a.part + (ps + row0 + r) * a.D + ds * S::DH : nullptr;
    });
  }
}

// Joins the splits of the forward: a block per row, 256 / W threads sharing
// each of the W >= D columns.  Bound by its launch and one read of the parts:
// 1920 rows of 256 in 4 splits, fp32, 6 us; 512 rows of 128 in 2 splits, 5 us.
template <class T, int W>
__global__ __launch_bounds__(256) void xattn_fwd_join(const XArgs a) {
  using E = typename T::elem;
  constexpr int P = 256 / W;
  __shared__ float part[256], top[P];
  const long long n = (long long)a.B * a.Hk * a.R, id = blockIdx.x;
  const int bh = (int)(id / a.R), r = (int)(id % a.R), lane = threadIdx.x % 64;
  const int d = threadIdx.x % W, p = threadIdx.x / W;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[2 * (s * n + id)]);
  m = wave_max(m);
  const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll 4
  for (int s = p; s < a.splits; s += P) {
    const float2 ml = *(const float2*)(a.part_ml + 2 * (s * n + id));
    const float f = __builtin_amdgcn_exp2f(ml.x - mu);
    l = fmaf(f, ml.y, l);
    if (d < a.D) o = fmaf(f, a.part[(s * n + id) * a.D + d], o);
  }
  if constexpr (P > 1) {
    part[threadIdx.x] = o;
    if (d == 0) top[p] = l;
    __syncthreads();
    if (p) return;
    o = l = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      o += part[i * W + d];
      l += top[i];
    }
  }
  const bool none = m == -INFINITY && l == 0.f;
  if (a.lse && d == 0) a.lse[id] = none ? INFINITY : x_lse<T>(m, l);
  if (d < a.D)
    x_row<E>(a.o, bh / a.Hk, bh % a.Hk, a.G, r)[d] = T::bits(none ? 0.f : o / l);
}

// ----------------------------------------------------------------- backward ---
// fp16 holds dS from 2^-24 to 2^16 only: dS is scaled by a power of two and the
// sum scaled back in fp32.  |dP| and |delta| are at most |dO| |V| in the 2-norm, of
// the row (for dK, whose sum runs over all rows, of the largest) and of the
// largest kept state, so |dS| <= 2 |dO| |V| =: b as P <= 1.  The scale and P's own
// bring b to [2^14, 2^15): nothing overflows, and dS keeps all of fp16's digits
// down to 2^-28 b.  (Following the largest dP from piece to piece instead spares the
// launch below, but costs registers: backward of 4 x 2048 rows on 2048 states,
// 16 heads of 128, 710 us against 541.)  bf16 and fp32 need none.
template <class T>
struct DownScale {
  static constexpr bool ON = std::is_same<T, XF16>::value;
  float v = 1.f;
  // dout: |dO|; square: of |V|
  __device__ __forceinline__ void set(float dout, float square) {
    const uint32_t e = (__float_as_uint(2.f * dout * sqrtf(square)) >> 23) & 255;
    if (ON && e != 0 && e != 255) v = __uint_as_float((254 - e) << 23);
  }
  __device__ __forceinline__ float operator()(float ds) const { return ON ? ds * v : ds; }
};

// The squares of the largest |V| of the kept states, a chunk of them per block.
// Bound by its launch, then by reading V once.  It adds to a backward: 2.5 us for
// 64 x 32 states of 4 heads of 64 (of 29), 5 for 3 x 777 of 3 heads of 80 (of 60),
// 7 for 4 x 1500 of 4 heads of 128 (of 266), 45 for 16 x 8192 of 8 (of 521).
template <class T, int DP>
__global__ __launch_bounds__(256) void xattn_vmax(const XArgs a) {
  using I = Img<T, DP>;
  using E = typename T::elem;
  constexpr int LANES = I::CPR, ROWS = 256 / LANES;
  __shared__ float top[4];
  const int bh = blockIdx.x / a.chunks, c = blockIdx.x % a.chunks, b = bh / a.Hk;
  const int lane = threadIdx.x % 64, ch = threadIdx.x % LANES;
  const int len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Tk) : a.Tk;
  const int per = (a.Tk + a.chunks - 1) / a.chunks;
  const int hi = (int)min((long long)len, (c + 1LL) * per);
  const E* V = (const E*)a.v.p + b * a.v.sb + bh % a.Hk * a.v.sh;
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  float x = 0.f;
#pragma unroll 4
  for (int j0 = c * per; j0 < hi; j0 += ROWS) {
    const int j = j0 + threadIdx.x / LANES;
    const bool in = j < hi && (!mask || mask[j]) && ch * I::E < a.D;
    const uint4 u = in ? ld_chunk<T>(V + j * a.v.st, ch, a.D) : zero16();
    E e[I::E];
    __builtin_memcpy(e, &u, 16);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < I::E; ++i) s = fmaf(T::val(e[i]), T::val(e[i]), s);
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) s += __shfl_xor(s, m);
    x = fmaxf(x, s);
  }
  x = wave_max(x);
  if (lane == 0) top[threadIdx.x / 64] = x;
  __syncthreads();
  if (threadIdx.x == 0) a.vmax[blockIdx.x] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// of all chunks of one key head, in every lane
__device__ __forceinline__ float x_vmax(const XArgs& a, int bh) {
  const int lane = threadIdx.x % 64;
  return wave_max(lane < a.chunks ? a.vmax[(long long)bh * a.chunks + lane] : 0.f);
}

// dQ of WR * 32 rows, streaming K and V; also delta (and fp16's |dO|) for
// xattn_dkv, which runs after it.  4 x 2048 rows on 2048 states, 16 heads of 128,
// bf16: 194 us, 1061 TFLOP/s, bound by the matrix units.  fp32, 64 x 30 rows on
// 196 states of 256: 20 us.
template <class T, int DP, int WR, int WS, int DS, int OCC>
__global__ __launch_bounds__(64 * WR * WS * DS) X_OCCUPANCY(OCC) void xattn_dq(const XArgs a) {
  using S = KeyStream<T, DP, WR, WS, DS, false>;
  using I = Img<T, S::DH>;
  using E = typename T::elem;
  const XWork w = x_work(a, a.q_lens, a.Tq, a.G, 32 * WR, a.kv_lens);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int wr = wave % WR, ws = wave / WR % WS, ds = wave / (WR * WS);
  const int lr = lane & 31, h = lane >> 5;
  const int rows = x_len(a.q_lens, w.b, a.Tq) * a.G;
  const int row0 = w.tile * WR * 32, row = row0 + wr * 32 + lr;
  const int len = row0 < rows ? x_len(a.kv_lens, w.b, a.Tk) : 0;
  int klo, khi;
  x_share(len, S::KT, a.splits, w.split, klo, khi);
  const float c2 = a.scale * LOG2E_X;
  const long long at = (long long)w.bh * a.R;

  const int Dh = a.D - ds * S::DH;           // columns from this wave's first on
  Rows32<T, S::DH> qf, df;
  float delta = 0.f, size = 0.f;
  {
    const bool live = row < rows;
    const E* o = live ? x_row<E>(a.o, w.b, w.g, a.G, row) + ds * S::DH : nullptr;
    Rows32<T, S::DH> of;
    qf.load(live ? x_row<E>(a.q, w.b, w.g, a.G, row) + ds * S::DH : nullptr, Dh, h);
    df.load(live ? x_row<E>(a.dout, w.b, w.g, a.G, row) + ds * S::DH : nullptr, Dh, h);
    of.load(o, Dh, h);
#pragma unroll
    for (int j = 0; j < I::NC; ++j) {
      const uint4 dv = df[j], ov = of[j];
      E x[I::E], y[I::E];
      __builtin_memcpy(x, &dv, 16);
      __builtin_memcpy(y, &ov, 16);
#pragma unroll
      for (int e = 0; e < I::E; ++e) {
        delta = fmaf(T::val(x[e]), T::val(y[e]), delta);
        if constexpr (DownScale<T>::ON) size = fmaf(T::val(x[e]), T::val(x[e]), size);
      }
    }
  }
  delta = xhalf_sum(delta);
  DownScale<T> down;
  if constexpr (DownScale<T>::ON) {
    size = sqrtf(xhalf_sum(size));
    down.set(size, x_vmax(a, w.bh));
  }
  if constexpr (DS > 1) {                      // of all columns
    lds_stf(4 * (wave * 32 + lr), delta);
    __syncthreads();
    delta = 0.f;
    for (int x = 0; x < DS; ++x) delta += lds_ldf(4 * (((x * WS + ws) * WR + wr) * 32 + lr));
    __syncthreads();
  }
  const float L = row < rows ? a.lse[at + row] : INFINITY;
  int turn = 0;

  auto masked = [&](f32x16 (&sp)[2], uint32_t kb) X_INLINE { x_mask(sp[0], kb, h); };
  constexpr int NB = S::DH / 32;
  f32x16 acc[NB] = {};
  // the scores of a piece in sp[0], dP in sp[1]; element(sp, e): their vector work
  auto run = [&](auto products, auto element) X_INLINE {
    S::run(a, w, klo, khi, ws, ds, masked,
           [&](auto first, auto rest, f32x16 (&sp)[2], const auto& ks, const auto&,
               f32x16 (&next)[2], const auto& kn, const auto& vn) X_INLINE {
      constexpr bool A = first.value, B = rest.value, P = decltype(products)::value;
      constexpr int RM = A ? 2 * I::NC : 0, TR = B && P ? I::NPF * NB : 0;
      uint4 p[I::NPF];
      if constexpr (A) next[0] = next[1] = f32x16{};
      x_step<RM, TR, S::AHEAD, OCC == 1 && DP <= 128>(
          [&](int i) X_INLINE { return i & 1 ? vn.rm(i / 2) : kn.rm(i / 2); },
          [&](int i, uint4 f) X_INLINE {
            next[i & 1] = T::mma(f, i & 1 ? df[i / 2] : qf[i / 2], next[i & 1]);
          },
          []() X_INLINE {},
          [&](int i) X_INLINE {
            if constexpr (B)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (e * RM / 16 == i) element(sp, e);
          },
          [&]() X_INLINE {
            if constexpr (B && !A)
#pragma unroll
              for (int e = 0; e < 16; ++e) element(sp, e);
            if constexpr (TR > 0)
#pragma unroll
              for (int c = 0; c < I::NPF; ++c) p[c] = I::pack(sp[0], c);
          },
          [&](int i) X_INLINE { return ks.tr(i / NB, i % NB); },
          [&](int i, uint4 f) X_INLINE { acc[i % NB] = T::mma(f, p[i / NB], acc[i % NB]); });
      if constexpr (A && !B) x_exchange<DS>(next, ws * WR + wr, ds, turn);
    });
  };
  auto probability = [&](float s) X_INLINE {             // times 2^PBITS
    return __builtin_amdgcn_exp2f(fmaf(s, c2, -L));
  };
  constexpr float POUT = 1.f / (1 << T::PBITS);
  // With few states, delta = sum P dP is summed from the products themselves:
  // dO . O carries the rounding of O to the type, which few states do not
  // average out (dQ was 1.53 times as far off as one rounding at 32 states,
  // against 1.42 times so).
  if (T::ES == 2 && a.Tk <= 64 && a.splits == 1) {
    float sum = 0.f;
    run(std::false_type{}, [&](f32x16 (&sp)[2], int e) X_INLINE {
      sum = fmaf(probability(sp[0][e]), sp[1][e], sum);
    });
    sum = xhalf_sum(sum);
    if constexpr (WS > 1) {
      __syncthreads();
      if (h == 0) lds_stf(4 * ((ws * WR + wr) * 32 + lr), sum);
      __syncthreads();
      sum = 0.f;
      for (int x = 0; x < WS; ++x) sum += lds_ldf(4 * ((x * WR + wr) * 32 + lr));
    }
    if (L != INFINITY) delta = sum * POUT;
  }
  if (w.split == 0 && ws == 0 && ds == 0 && h == 0 && row < a.R) {
    a.delta[at + row] = delta;
    if constexpr (DownScale<T>::ON) a.size[at + row] = size;
  }
  run(std::true_type{}, [&](f32x16 (&sp)[2], int e) X_INLINE {
    sp[0][e] = down(probability(sp[0][e]) * (sp[1][e] - delta));
  });
  const float mul = a.scale * POUT / down.v;
  const bool none = L == INFINITY;
  const int tid = threadIdx.x % (64 * WR * WS);
  if (a.splits == 1) {
    x_store<T, S::DH, WR, WS>(acc, mul, none, Dh, tid, ds * S::OUT, [&](int r) -> E* {
      return row0 + r < a.R ? x_row<E>(a.dq, w.b, w.g, a.G, row0 + r) + ds * S::DH : nullptr;
    });
  } else {
    const long long ps = ((long long)w.split * a.B * a.Hk + w.bh) * a.R;
    x_store<XF32, S::DH, WR, WS>(acc, mul, none, Dh, tid, ds * S::OUT32, [&](int r) -> float* {
      return row0 + r < a.R ? a.part + (ps + row0 + r) * a.D + ds * S::DH : nullptr;
    });
  }
}

// dK and dV of WC * 32 states, streaming Q and dO, 32 WS rows at a time; WS
// waves share the states and take different rows, DS waves the columns of the
// results: of fp32 as above, of 16-bit types past 128 columns because both
// accumulators are too large for one wave's registers (each of the two forms
// all of the scores, 6 products where 4 would do).
//
// 4 x 2048 rows on 2048 states, 16 heads of 128, bf16: 290 us, 946 TFLOP/s.
// A wave of 128 columns is alone on its SIMD and issues 320 instructions a
// piece in the time of 32 matrix instructions and half as long again: bound by
// issue.  fp32, 64 x 30 rows on 196 states of 256: 26 us, 30 TFLOP/s (36 with the
// rows that fill the last pieces).
template <class T, int DP, int WC, int WS, int DS>
struct DkvCfg {
  static constexpr int NT = 64 * WC * WS * DS, RT = 32 * WS;
  static constexpr int AHEAD = T::ES == 4 ? 8 : DP == 128 ? 6 : 4;
  static constexpr bool MEM = T::ES == 4;
  static constexpr int TILE = MEM ? 0 : 2 * Img<T, DP>::bytes(RT) + 8 * RT;   // Q, dO, L, delta
  static constexpr int FED = MEM ? (DS > 1 ? 2 * 8192 * WC * WS * DS : 0) : 4 * TILE;
  static constexpr int OUT = x_store_bytes<T, DP / DS, WC, WS>();
  static constexpr int OUT32 = x_store_bytes<XF32, DP / DS, WC, WS>();
  static constexpr int LDS = x_max(x_max(FED, DS * OUT), 64);
  static constexpr int LDS32 = x_max(LDS, DS * OUT32);
};

template <class T, int DP, int WC, int WS, int DS, int OCC>
__global__ __launch_bounds__(64 * WC * WS * DS) X_OCCUPANCY(OCC) void xattn_dkv(const XArgs a) {
  using C = DkvCfg<T, DP, WC, WS, DS>;
  constexpr int RT = C::RT;
  // operands: a wave's own columns (fp32) or all
  constexpr int DH = DP / DS, NB = DH / 32, DO = C::MEM ? DH : DP;
  using I = Img<T, DO>;
  using E = typename T::elem;
  const XWork w = x_work(a, a.kv_lens, a.Tk, 1, 32 * WC, a.q_lens);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int wc = wave % WC, ws = wave / WC % WS, ds = wave / (WC * WS);
  const int lr = lane & 31, h = lane >> 5;
  const int len = x_len(a.kv_lens, w.b, a.Tk);
  const int key0 = w.tile * WC * 32, key = key0 + wc * 32 + lr;
  const int rows = x_len(a.q_lens, w.b, a.Tq) * a.G;
  int rlo, rhi;
  x_share(key0 < len ? rows : 0, RT, a.splits, w.split, rlo, rhi);
  const bool kept = key < len && (!a.mask || a.mask[w.b * a.mask_sb + key]);
  const float c2 = a.scale * LOG2E_X;
  const long long at = (long long)w.bh * a.R;

  DownScale<T> down;
  if constexpr (DownScale<T>::ON) {
    float x = 0.f;
    for (int r = threadIdx.x; r < rows; r += C::NT) x = fmaxf(x, a.size[at + r]);
    x = wave_max(x);
    if (lane == 0) lds_stf(4 * wave, x);
    __syncthreads();
    for (int i = 0; i < C::NT / 64; ++i) x = fmaxf(x, lds_ldf(4 * i));
    down.set(x, x_vmax(a, w.bh));
    __syncthreads();
  }

  const int c0 = C::MEM ? ds * DH : 0;         // first column of the operands
  Rows32<T, DO> kf, vf;
  const uint32_t kept32 = (uint32_t)__ballot(kept);     // (both halves: the same states)
  auto own = [&]() X_INLINE {
    if constexpr (C::MEM) {
      const uint32_t kst = (uint32_t)a.k.st * 4, vst = (uint32_t)a.v.st * 4;
      auto at_k = [=](int r) X_INLINE { return r * kst; };
      auto at_v = [=](int r) X_INLINE { return r * vst; };
      const int k0 = key0 + 32 * wc;
      const MemSrc<DO, T::VEC, decltype(at_k)> ks(x_key<E>(a.k, w.b, w.g, k0) + c0, at_k, kept32,
                                                  lane, a.D - c0);
      const MemSrc<DO, T::VEC, decltype(at_v)> vs(x_key<E>(a.v, w.b, w.g, k0) + c0, at_v, kept32,
                                                  lane, a.D - c0);
#pragma unroll
      for (int j = 0; j < I::NC; ++j) {
        kf.f[j] = ks.rm(j);
        vf.f[j] = vs.rm(j);
      }
    } else {
      kf.load(kept ? x_key<E>(a.k, w.b, w.g, key) : nullptr, a.D, h);
      vf.load(kept ? x_key<E>(a.v, w.b, w.g, key) : nullptr, a.D, h);
    }
  };
  if constexpr (!C::MEM) own();
  f32x16 dk[NB] = {}, dv[NB] = {};
  int turn = 0;

  // A step as x_step runs it: scores and dP of `next` beside the rest of sp, a
  // piece of 32 rows; lse(k), del(k): L and delta of its rows acc_row(4 k + e, h)
  auto work = [&](auto first, auto rest, f32x16 (&sp)[2], const auto& qs, const auto& os, auto lse,
                  auto del, f32x16 (&next)[2], const auto& qn, const auto& on) X_INLINE {
    constexpr bool A = first.value, B = rest.value;
    constexpr int RM = A ? 2 * I::NC : 0, TR = B ? 2 * I::NPF * NB : 0;
    const int b0 = C::MEM ? 0 : ds * NB;
    f32x4 L[4], t[4];
    uint4 p[I::NPF], g[I::NPF];
    auto element = [&](int i) X_INLINE {
      sp[0][i] = __builtin_amdgcn_exp2f(fmaf(sp[0][i], c2, -L[i / 4][i % 4]));
      sp[1][i] = down(sp[0][i] * (sp[1][i] - t[i / 4][i % 4]));
    };
    auto pack = [&](int c) X_INLINE {
      p[c] = I::pack(sp[0], c);
      g[c] = I::pack(sp[1], c);
    };
    if constexpr (A) next[0] = next[1] = f32x16{};
    x_step<RM, TR, C::AHEAD, OCC == 1>(
        [&](int i) X_INLINE { return i & 1 ? on.rm(i / 2) : qn.rm(i / 2); },
        [&](int i, uint4 f) X_INLINE {
          next[i & 1] = T::mma(f, i & 1 ? vf[i / 2] : kf[i / 2], next[i & 1]);
        },
        [&]() X_INLINE {
          if constexpr (B)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              L[k] = lse(k);
              t[k] = del(k);
            }
        },
        [&](int i) X_INLINE {
          if constexpr (B) {
            if (i == RM / 2 && I::NPF == 2) pack(0);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e * RM / 16 == i) element(e);
          }
        },
        [&]() X_INLINE {
          if constexpr (B) {
            if constexpr (!A)
#pragma unroll
              for (int e = 0; e < 16; ++e) element(e);
#pragma unroll
            for (int c = A && I::NPF == 2 ? 1 : 0; c < I::NPF; ++c) pack(c);
          }
        },
        [&](int i) X_INLINE {
          const int c = i / 2 / NB, db = i / 2 % NB;
          return i & 1 ? qs.tr(c, b0 + db) : os.tr(c, b0 + db);
        },
        [&](int i, uint4 f) X_INLINE {
          const int c = i / 2 / NB, db = i / 2 % NB;
          if (i & 1)
            dk[db] = T::mma(f, g[c], dk[db]);
          else
            dv[db] = T::mma(f, p[c], dv[db]);
        });
    if constexpr (C::MEM && A && !B) x_exchange<DS>(next, ws * WC + wc, ds, turn);
  };
  using Yes = std::true_type;
  using No = std::false_type;
  // byte offset of row i of a tile that begins with a token's first head
  auto in_tile = [&](const XView& v) {
    const uint32_t st = (uint32_t)v.st * T::ES, sh = (uint32_t)v.sh * T::ES;
    const uint32_t G = a.G, per = a.per_g, one = G == 1 ? ~0u : 0u;
    return [=](uint32_t i) X_INLINE -> uint32_t {
      const uint32_t t = __umulhi(i, per) + (i & one);       // i / G, i G < 2^32
      return t * st + (i - t * G) * sh;
    };
  };
  if constexpr (C::MEM) {
    for (int t = rlo; t < rhi; t += RT) {
      const int r0 = t + 32 * ws, n = rhi - r0;
      const uint32_t live = n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1 : 0u;
      if (DS == 1 && !live) continue;
      // offsets from the first row's token
      const int t0 = a.G == 1 ? r0 : (int)((unsigned)r0 / (unsigned)a.G), g0 = r0 - t0 * a.G;
      const auto qo = in_tile(a.q), oo = in_tile(a.dout);
      auto at_q = [=](int i) X_INLINE { return qo(g0 + i); };
      auto at_o = [=](int i) X_INLINE { return oo(g0 + i); };
      MemSrc<DO, T::VEC, decltype(at_q)> qs(x_row<E>(a.q, w.b, w.g, a.G, t0 * a.G) + c0, at_q, live,
                                            lane, a.D - c0);
      MemSrc<DO, T::VEC, decltype(at_o)> os(x_row<E>(a.dout, w.b, w.g, a.G, t0 * a.G) + c0, at_o,
                                            live, lane, a.D - c0);
      asm volatile("" ::: "memory");
      own();            // again for each piece: held over all, they would cost a wave per SIMD
      f32x16 sp[2];
      f32x4 L[4], delta[4];            // read before the products that they wait beside
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = acc_row(i, h);
        const long long j = at + min(r0 + r, rhi - 1);         // no branch
        const float x = a.lse[j], y = a.delta[j];
        L[i / 4][i % 4] = r < n ? x : INFINITY;
        delta[i / 4][i % 4] = r < n ? y : 0.f;
      }
      auto lse = [&](int k) X_INLINE { return L[k]; };
      auto del = [&](int k) X_INLINE { return delta[k]; };
      work(Yes{}, No{}, sp, qs, os, lse, del, sp, qs, os);
      __builtin_amdgcn_sched_barrier(0);
      qs.open();
      os.open();
      work(No{}, Yes{}, sp, qs, os, lse, del, sp, qs, os);
    }
  } else {
    constexpr uint32_t D0 = I::bytes(RT), L0 = 2 * D0, T0 = L0 + 4 * RT;
    using F = Feed<T, DP, RT, C::NT>;
    constexpr int STATS = 2 * RT / 64;                // instructions for L and delta
    F fq, fd;
    fq.init(in_tile(a.q), a.D);
    fd.init(in_tile(a.dout), a.D);
    __syncthreads();
    for (int i = 0; i < 4; ++i) {
      fq.clear(i * C::TILE);
      fd.clear(i * C::TILE + D0);
    }
    const int np = (rhi - rlo + RT - 1) / RT, full = (rhi - rlo) / RT;
    // L and delta of a tile, one after the other; every wave fetches them (the
    // same values to the same places), so that all count the same instructions
    const float* stat_at[STATS];
#pragma unroll
    for (int i = 0; i < STATS; ++i) {
      const int j = 64 * i + lane;
      stat_at[i] = (j < RT ? a.lse : a.delta) + at + rlo + j % RT;
    }
    auto stats = [&](int n, uint32_t l0, auto plain) X_INLINE {
#pragma unroll
      for (int i = 0; i < STATS; ++i) {
        const int j = 64 * i + lane;
        const float* p = stat_at[i] + n * RT;
        if constexpr (!plain.value)
          if (rlo + n * RT + j % RT >= rhi) p = j < RT ? x_pad + 4 : x_pad;
        dma4(p, l0 + L0 + 256 * i);
      }
    };
    // a tile's first row, where G, a power of two, divides RT
    const int sh = 31 - __builtin_clz(a.G);
    auto first = [&](const XView& v, int r0) -> const E* {
      return x_row<E>(v, w.b, w.g, a.G, 0) + (long long)(r0 >> sh) * v.st;
    };
    auto feed = [&](int n) X_INLINE {
      const int r0 = rlo + n * RT;
      const uint32_t l0 = (n & 3) * C::TILE;
      if (n >= np) return;
      stats(n, l0, No{});
      auto kept = [&](int r) X_INLINE { return r0 + r < rhi; };
      if (!a.fast_q) {
        auto row = [&](const XView& v) X_INLINE {
          return [&](int r) X_INLINE {
            return kept(r) ? x_row<E>(v, w.b, w.g, a.G, r0 + r) : nullptr;
          };
        };
        fq.copy(row(a.q), a.D, l0);
        fd.copy(row(a.dout), a.D, l0 + D0);
      } else if (n < full) {
        fq.start(first(a.q, r0), l0);
        fd.start(first(a.dout, r0), l0 + D0);
      } else {
        fq.start_kept(first(a.q, r0), kept, l0);
        fd.start_kept(first(a.dout, r0), kept, l0 + D0);
      }
    };
    feed(0);
    feed(1);
    feed(2);
    auto wait = [&](int n, auto plain) X_INLINE {
      if constexpr (plain.value) {
        ring_barrier<2 * F::N + STATS>();
        const int r0 = rlo + (n + 3) * RT;
        const uint32_t l0 = ((n + 3) & 3) * C::TILE;
        stats(n + 3, l0, Yes{});
        fq.start(first(a.q, r0), l0);
        fd.start(first(a.dout, r0), l0 + D0);
      } else {
        if (a.fast_q && n >= 0 && n + 2 < np)
          ring_barrier<2 * F::N + STATS>();
        else
          ring_barrier<0>();
        if (n >= 0) feed(n + 3);
      }
    };
    const uint32_t mine = I::bytes(32) * ws;
    auto src = [&](uint32_t l0) { return LdsSrc<T, DP>{l0 + mine, lane}; };
    auto stat = [&](int slot, uint32_t what) X_INLINE {
      return [=](int k) X_INLINE {
        return __builtin_bit_cast(
            f32x4, lds_ld16(slot * C::TILE + what + 4 * (32 * ws + 8 * k + 4 * h)));
      };
    };
    auto Q_ = [&](int slot) X_INLINE { return src(slot * C::TILE); };
    auto O_ = [&](int slot) X_INLINE { return src(slot * C::TILE + D0); };
    x_pipe<2>(
        np, a.fast_q ? full - 3 : 0, wait,
        [&](f32x16 (&sp)[2], int s) X_INLINE {
          work(Yes{}, No{}, sp, Q_(s), O_(s), stat(s, L0), stat(s, T0), sp, Q_(s), O_(s));
        },
        [](f32x16 (&)[2], int, auto) {},
        [&](f32x16 (&sp)[2], int s, f32x16 (&next)[2], int t) X_INLINE {
          work(Yes{}, Yes{}, sp, Q_(s), O_(s), stat(s, L0), stat(s, T0), next, Q_(t), O_(t));
        },
        [&](f32x16 (&sp)[2], int s) X_INLINE {
          work(No{}, Yes{}, sp, Q_(s), O_(s), stat(s, L0), stat(s, T0), sp, Q_(s), O_(s));
        });
  }
  const int tid = threadIdx.x % (64 * WC * WS), Dh = min(a.D - ds * DH, DH);
  constexpr float POUT = 1.f / (1 << T::PBITS);
  const float mul = a.scale * POUT / down.v;
  if (a.splits == 1) {
    const auto dst = [&](const XView& v) {
      return [&](int r) -> E* {
        return key0 + r < a.Tk ? x_key<E>(v, w.b, w.g, key0 + r) + ds * DH : nullptr;
      };
    };
    x_store<T, DH, WC, WS>(dk, mul, !kept, Dh, tid, ds * C::OUT, dst(a.dk));
    x_store<T, DH, WC, WS>(dv, POUT, !kept, Dh, tid, ds * C::OUT, dst(a.dv));
  } else {
    const auto dst = [&](int which) {
      const long long ps =
          (((long long)which * a.splits + w.split) * a.B * a.Hk + w.bh) * a.Tk + key0;
      return [=](int r) -> float* {
        return key0 + r < a.Tk ? a.part + (ps + r) * a.D + ds * DH : nullptr;
      };
    };
    x_store<XF32, DH, WC, WS>(dk, mul, !kept, Dh, tid, ds * C::OUT32, dst(0));
    x_store<XF32, DH, WC, WS>(dv, POUT, !kept, Dh, tid, ds * C::OUT32, dst(1));
  }
}

// Sums the splits of a gradient, as the forward's are joined: dQ (R rows), or
// dK and dV (blockIdx.y; Tk rows).
template <class T, int W, bool KV>
__global__ __launch_bounds__(256) void xattn_join(const XArgs a) {
  using E = typename T::elem;
  constexpr int P = 256 / W;
  __shared__ float sum[256];
  const int per = KV ? a.Tk : a.R;
  const long long n = (long long)a.B * a.Hk * per, id = blockIdx.x;
  const int bh = (int)(id / per), r = (int)(id % per), b = bh / a.Hk, g = bh % a.Hk;
  const int d = threadIdx.x % W, p = threadIdx.x / W;
  const float* part = a.part + (KV ? blockIdx.y * a.splits * n * a.D : 0);
  float x = 0.f;
  if (d < a.D) {
#pragma unroll 4
    for (int s = p; s < a.splits; s += P) x += part[(s * n + id) * a.D + d];
  }
  if constexpr (P > 1) {
    sum[threadIdx.x] = x;
    __syncthreads();
    if (p) return;
    x = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) x += sum[i * W + d];
  }
  E* to = KV ? x_key<E>(blockIdx.y ? a.dv : a.dk, b, g, r) : x_row<E>(a.dq, b, g, a.G, r);
  if (d < a.D) to[d] = T::bits(x);
}

// ------------------------------------------------------------------- launch ---
enum { X_FWD, X_DQ, X_DKV };

struct XPlan {
  int waves, tiles, splits;      // waves that own rows (dK, dV: states), 32 each
};
// Waves along the columns: fp32 64 columns each; dK, dV of 16-bit types two
// waves past 128 columns (at 128, one wave of 32 products a piece, alone on its
// SIMD, took 149 us where two of 24 took 166: 4 x 1024 rows, 16 heads on 4, on
// 1500 states).
constexpr int x_columns(int type, int what, int dp) {
  return type == 1 ? dp / 64 : what == X_DKV && dp > 128 ? 2 : 1;
}
// Least waves that own rows (states): the rings of fewer would pass the LDS, or
// of 64 columns leave a CU one block instead of two (4 x 5 x 1500, 12 heads,
// masked: 13.3 us against 15.0 at each one's best splits).
constexpr int x_least(int type, int what, int dp) {
  if (type == 1 || (dp == 64 && what == X_DKV)) return 1;
  return dp <= 128 || what == X_DKV ? 2 : 4;
}
// The split of one kernel's work.  `own` rows (dK, dV: states) belong to the
// waves, the others are streamed.  A block's four waves (or those that the
// columns leave) own 32 rows each while that gives every CU a block; below,
// two or all of them share rows and take different parts of the stream, where
// that has a piece of 32 for each (1 x 2048 x 2048 of 8 heads on one: 38 us
// against 48; 8 x 64 x 512, 8 heads of 64: 10.0 against 12.8); not for a few rows
// of 128 columns under a mask, whose steps take longer than their tiles, where
// the splits fill the card by themselves, two blocks to a CU (16 x 1 x 8192, 32
// heads on 8: 101 us against 142; without a mask 84 against 77).  What still leaves
// CUs without a block splits the stream over blocks, 128 items (fp32: 64) or
// more each and no more blocks than run at once; a second launch joins them
// (17 tokens of 8 heads on 8192 states: 32 us against 114; not at 99 blocks, 3 x
// 333 x 777, 6 heads of 80 on 3, masked: 31 us both ways; 4 x 5 x 1500, 12 heads of 64, masked: 14.4 us in one round of 480
// blocks, 21.7 in one and an eighth of 256; 64 x 30 x 196 of 256, fp32: 21.2 us by 4
// splits, 23.0 by 7).
inline XPlan x_plan(const XArgs& a, int type, int what) {
  const int own = what == X_DKV ? a.Tk : a.R, stream = what == X_DKV ? a.R : a.Tk;
  const long long heads = (long long)a.B * a.Hk;
  const int dp = a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256, all = 4 / x_columns(type, what, dp);
  const bool masked = a.mask && dp == 128 && what != X_DKV;
  XPlan p;
  for (p.waves = all;; p.waves /= 2) {
    p.tiles = (own + 32 * p.waves - 1) / (32 * p.waves);
    if (p.waves == x_least(type, what, dp) || p.tiles * heads >= 256 ||
        stream <= 32 * (all / p.waves) || (masked && own <= 32 && heads >= 96))
      break;
  }
  const long long blocks = p.tiles * heads;
  const int each = type == 1 ? 64 : 128, most = (stream + each - 1) / each;
  // blocks at once: two per CU where their rings leave room
  // (dK, dV join twice as much: 64 x 196 rows on 32 states, 4 heads of 64, 14 us
  // unsplit, 16 + 11 in two)
  const bool two = type == 1 || (what != X_DKV && ((dp == 64 && p.waves > 1) ||
                                                   (dp == 128 && p.waves == 4)));
  const int slots = two ? 512 : 256;
  const long long want = blocks >= (own <= 32 ? slots : 96) ? 1 : slots / blocks;
  p.splits = (int)(want < most ? want : most);
  return p;
}

// Blocks for the largest |V| of a key head: 32 states or more each, no more than
// 2048 in all where there are not more heads, at most one per lane of a wave.
inline int x_chunks_of_v(const XArgs& a) {
  const long long most = (a.Tk + 31) / 32, want = 2048 / ((long long)a.B * a.Hk);
  const long long n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

// threads of a launch
constexpr long long X_THREADS = 0xffffffffLL;

template <class K>
int x_go(K kernel, const XArgs& a, int lds, int nt, void* stream) {
  if (lds > 64 * 1024)
    if (const int e = set_max_lds((const void*)kernel, lds)) return e;
  const long long grid = (long long)a.tiles * a.splits * a.B * a.Hk;
  if (grid * nt > X_THREADS) return 1001;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(nt), lds, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

template <class T, int DP, int W, bool FWD>
int x_rows(const XArgs& a, void* stream) {
  constexpr int DS = x_columns(T::TYPE, X_FWD, DP), WS = 4 / DS / W;
  constexpr int OCC = T::ES == 4 || DP * (4 / W) <= 128 ? 2 : 1;        // rings of 64 KiB
  using S = KeyStream<T, DP, W, WS, DS, FWD>;
  const int lds = a.splits > 1 ? S::LDS32 : S::LDS;
  if constexpr (FWD)
    return x_go(xattn_fwd<T, DP, W, WS, DS, OCC>, a, lds, S::NT, stream);
  else
    return x_go(xattn_dq<T, DP, W, WS, DS, OCC>, a, lds, S::NT, stream);
}
template <class T, int DP, int W>
int x_states(const XArgs& a, void* stream) {
  constexpr int DS = x_columns(T::TYPE, X_DKV, DP), WS = 4 / DS / W;
  using C = DkvCfg<T, DP, W, WS, DS>;
  constexpr int OCC = T::ES == 4 || (DP <= 64 && C::FED <= 80 * 1024) ? 2 : 1;
  return x_go(xattn_dkv<T, DP, W, WS, DS, OCC>, a, a.splits > 1 ? C::LDS32 : C::LDS, C::NT, stream);
}
template <class T, int DP, int W>
int x_waves(const XArgs& a, int waves, int what, void* stream) {
  if constexpr (W > 1)
    if (waves < W) return x_waves<T, DP, W / 2>(a, waves, what, stream);
  constexpr auto takes = [](int k) {
    return W * x_columns(T::TYPE, k, DP) <= 4 && W >= x_least(T::TYPE, k, DP);
  };
  if constexpr (takes(X_FWD))
    if (what == X_FWD) return x_rows<T, DP, W, true>(a, stream);
  if constexpr (takes(X_DQ))
    if (what == X_DQ) return x_rows<T, DP, W, false>(a, stream);
  if constexpr (takes(X_DKV))
    if (what == X_DKV) return x_states<T, DP, W>(a, stream);
  return 1001;
}

template <class T, int DP>
int x_run(XArgs a, int what, void* stream) {
  const XPlan p = x_plan(a, T::TYPE, what);
  a.tiles = p.tiles;
  a.splits = p.splits;
  if constexpr (DownScale<T>::ON)
    if (what == X_DQ)
      hipLaunchKernelGGL((xattn_vmax<T, DP>), dim3((unsigned)(a.B * a.Hk * a.chunks)), dim3(256), 0,
                         (hipStream_t)stream, a);
  const int e = x_waves<T, DP, 4>(a, p.waves, what, stream);
  if (e || a.splits == 1) return e;
  const dim3 grid((unsigned)(a.B * a.Hk * (what == X_DKV ? a.Tk : a.R)), what == X_DKV ? 2 : 1);
  if (what == X_FWD)
    hipLaunchKernelGGL((xattn_fwd_join<T, DP>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else if (what == X_DQ)
    hipLaunchKernelGGL((xattn_join<T, DP, false>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((xattn_join<T, DP, true>), grid, dim3(256), 0, (hipStream_t)stream, a);
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
