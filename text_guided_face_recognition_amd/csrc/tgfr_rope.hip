// RMS norm of each head of the queries and keys with the position rotation in
// the same pass, forward and backward (gfx950).
//
//   n = x rsqrt(mean_d x^2 + eps);  u = n w
//   (ya, yb) = (ua cos t - ub sin t, ub cos t + ua sin t) for the R / 2 pairs
//   of a head: (i, i + R / 2), or (2 i, 2 i + 1) when interleaved; the D - R
//   elements behind them are normed only.
//   t = pos f_i, f_i = base^(-i / pairs).  With more position axes (a grid of
//   regions) the pairs fall into equal runs, one per axis.
// Backward, with du = dy rotated by -t:
//   dw = sum du n;  dn = du w;  dx = r (dn - n mean_d(dn n))
//
// The angle: f_i / 2 pi is given as a 64-bit fraction of a turn, so pos times
// it in 64-bit integers drops whole turns exactly, for any position; the
// fraction's own rounding makes the angle off by at most pos 2^-65 turns.
//
// Bound by memory: x is read once and y written once, 16 bytes per lane and
// load, LPR lanes per head.  A wave takes one token, or as many as fill it
// where heads are few; its lanes form the sines of the tokens' pairs once, each
// another one, and share them through LDS (formed by each lane for itself,
// they took more vector instructions than all the rest).  4 x 4096 tokens of 32
// + 8 heads of 128, bf16: 75 us, 4.5 TB/s (a copy: 4.7).  Backward of 2 x 4096 of
// them: 70 us, 3.6 TB/s, three streams and the partial sums of dw, whose second
// launch takes 5 us.
#include "tgfr_common.h"

using namespace tgfr;

namespace {

struct NPart {
  const void* x;        // input [B][T][H][D], strides in elements
  long long xb, xt, xh;
  const void* dy;       // backward: gradient of y
  long long gb, gt, gh;
  void* y;              // y, or dx; strides as given
  long long yb, yt, yh;
  const float* w;       // [D]
  const void* pos;      // positions; NULL: 0 .. T - 1 on every axis
  long long pb, pt, pa;
  int B, T, H;
  int lg;               // 2^lg >= min(H, 64 / LPR) heads of a token side by side
  int blocks;           // of this part
};
struct NArgs {
  NPart p[2];
  const unsigned long long* turn;   // [R / 2]
  float* part;          // backward: [blocks][D] partial dw
  int D, R, per, interleaved, pos32;
  int many;             // a unit takes all heads of its tokens
  float eps;
};

template <int K>
struct Num;
template <>
struct Num<0> {   // bf16
  using E = uint16_t;
  static __device__ __forceinline__ float val(E u) { return bf_val(u); }
  static __device__ __forceinline__ E bits(float x) { return bf_bits(x); }
};
template <>
struct Num<1> {   // fp32
  using E = float;
  static __device__ __forceinline__ float val(E u) { return u; }
  static __device__ __forceinline__ E bits(float x) { return x; }
};
template <>
struct Num<2> {   // fp16
  using E = uint16_t;
  static __device__ __forceinline__ float val(E u) {
    return (float)__builtin_bit_cast(_Float16, u);
  }
  static __device__ __forceinline__ E bits(float x) { return f16_bits(x); }
};

// V values at an address aligned to the element only
template <class E, int V>
struct __attribute__((packed, aligned(sizeof(E)))) Pack {
  E e[V];
};

// Where a lane's V pairs lie.  Chunked loads need them in one piece: the
// elements a0 .. and b0 .. (or 2 V from a0 on, interleaved).
__device__ __forceinline__ int n_first(const NArgs& a, int p) {
  if (a.interleaved) return 2 * p;
  return p < a.R / 2 ? p : a.R + (p - a.R / 2);
}
__device__ __forceinline__ int n_second(const NArgs& a, int p) {
  if (a.interleaved) return 2 * p + 1;
  return p < a.R / 2 ? p + a.R / 2 : a.R + (p - a.R / 2) + (a.D - a.R) / 2;
}

// V pairs of a row of D elements: u[0 .. V) the first, u[V .. 2V) the second
template <int K, int V, bool CH>
__device__ __forceinline__ void n_load(const NArgs& a, const void* base, int p0, float (&u)[2 * V]) {
  using E = typename Num<K>::E;
  const E* x = (const E*)base;
  if constexpr (CH) {
    Pack<E, V> l, r;
    l = *(const Pack<E, V>*)(x + n_first(a, p0));
    r = *(const Pack<E, V>*)(x + (a.interleaved ? 2 * p0 + V : n_second(a, p0)));
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        u[i] = Num<K>::val(2 * i < V ? l.e[2 * i] : r.e[2 * i - V]);
        u[V + i] = Num<K>::val(2 * i + 1 < V ? l.e[2 * i + 1] : r.e[2 * i + 1 - V]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        u[i] = Num<K>::val(l.e[i]);
        u[V + i] = Num<K>::val(r.e[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool in = p0 + i < a.D / 2;
      u[i] = in ? Num<K>::val(x[n_first(a, p0 + i)]) : 0.f;
      u[V + i] = in ? Num<K>::val(x[n_second(a, p0 + i)]) : 0.f;
    }
  }
}
template <int K, int V, bool CH>
__device__ __forceinline__ void n_store(const NArgs& a, void* base, int p0,
                                        const float (&u)[2 * V]) {
  using E = typename Num<K>::E;
  E* y = (E*)base;
  if constexpr (CH) {
    Pack<E, V> l, r;
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        (2 * i < V ? l.e[2 * i] : r.e[2 * i - V]) = Num<K>::bits(u[i]);
        (2 * i + 1 < V ? l.e[2 * i + 1] : r.e[2 * i + 1 - V]) = Num<K>::bits(u[V + i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        l.e[i] = Num<K>::bits(u[i]);
        r.e[i] = Num<K>::bits(u[V + i]);
      }
    }
    *(Pack<E, V>*)(y + n_first(a, p0)) = l;
    *(Pack<E, V>*)(y + (a.interleaved ? 2 * p0 + V : n_second(a, p0))) = r;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (p0 + i < a.D / 2) {
        y[n_first(a, p0 + i)] = Num<K>::bits(u[i]);
        y[n_second(a, p0 + i)] = Num<K>::bits(u[V + i]);
      }
  }
}

template <int LPR>
__device__ __forceinline__ float n_sum(float v) {
  if constexpr (LPR >= 64) v = xhalf_sum(v);
  if constexpr (LPR >= 32) v = x16_sum(v);
  if constexpr (LPR >= 16) v += dpp<0x140>(v);
  if constexpr (LPR >= 8) v += dpp<0x141>(v);
  v += dpp<0xB1>(v);
  return v + dpp<0x4E>(v);
}

// A wave's unit: 64 / LPR >> lg tokens, and 2^lg of their heads at once.
template <int V, int LPR>
struct Unit {
  static constexpr int HPW = 64 / LPR;
  int h0, h1, step;          // this lane's heads: h0, h0 + step, ... below h1
  int b, t;                  // its token (valid: it has one)
  bool valid;

  static __device__ __forceinline__ long long count(const NArgs& a, const NPart& q) {
    const long long tokens = (long long)q.B * q.T, at_once = HPW >> q.lg;
    return (tokens + at_once - 1) / at_once * (a.many ? 1 : (q.H + (1 << q.lg) - 1) >> q.lg);
  }
  static __device__ __forceinline__ void token(const NPart& q, int id, int& b, int& t) {
    b = (unsigned)id / (unsigned)q.T;
    t = id - b * q.T;
  }
  // sc: LDS of the wave, V * 64 pairs (sine, cosine)
  __device__ __forceinline__ Unit(const NArgs& a, const NPart& q, long long unit, float2* sc) {
    const int lane = threadIdx.x % 64, g = lane / LPR;
    const int hu = a.many ? 1 : (q.H + (1 << q.lg) - 1) >> q.lg;
    const int tg = hu == 1 ? (int)unit : (int)(unit / hu), hc = (int)(unit - (long long)tg * hu);
    const int tokens = q.B * q.T, first = tg * (HPW >> q.lg);
    step = 1 << q.lg;
    h0 = hc * step + (g & (step - 1));
    h1 = a.many ? q.H : min(q.H, (hc + 1) * step);
    valid = first + (g >> q.lg) < tokens;
    token(q, min(first + (g >> q.lg), tokens - 1), b, t);
    asm volatile("" ::: "memory");                    // the last unit's are read
    // Sines: 64 / (tokens of the wave) lanes per token, pair after pair.
    const int per = LPR << q.lg;                      // lanes per token
    int sb, st;
    token(q, min(first + lane / per, tokens - 1), sb, st);
    for (int p = lane & (per - 1); p < LPR * V; p += per) {
      float2 v = make_float2(0.f, 1.f);
      if (p < a.R / 2) {
        long long at = st;
        if (q.pos) {
          const long long i = sb * q.pb + st * q.pt + (a.per == a.R / 2 ? 0 : p / a.per) * q.pa;
          at = a.pos32 ? ((const int*)q.pos)[i] : ((const long long*)q.pos)[i];
        }
        const unsigned long long f = (unsigned long long)at * a.turn[p];
        // signed fraction of a turn, [-1/2, 1/2)
        const float turns =
            fmaf((float)(uint32_t)f, 0x1p-64f, (float)(int32_t)(f >> 32) * 0x1p-32f);
        sincospif(2.f * turns, &v.x, &v.y);
      }
      sc[lane / per * (LPR * V) + p] = v;
    }
    asm volatile("" ::: "memory");                    // (one wave's LDS is in order)
  }
  __device__ __forceinline__ void sines(const NPart& q, const float2* sc, float (&sn)[V],
                                        float (&cs)[V]) const {
    const int lane = threadIdx.x % 64, c = lane % LPR, g = lane / LPR;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 v = sc[(g >> q.lg) * (LPR * V) + c * V + i];
      sn[i] = v.x;
      cs[i] = v.y;
    }
  }
};

// this block's part, and its place among that part's blocks
__device__ __forceinline__ int n_part(const NArgs& a, int& blk) {
  const int k = (int)blockIdx.x >= a.p[0].blocks;
  blk = k ? blockIdx.x - a.p[0].blocks : blockIdx.x;
  return k;
}

template <int KI, int KO, int V, int LPR, bool CH>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const NArgs a) {
  __shared__ float2 sc[4][64 * V];
  using U = Unit<V, LPR>;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, p0 = lane % LPR * V;
  int blk;
  const NPart& q = a.p[n_part(a, blk)];
  const bool in = p0 < a.D / 2;
  using EI = typename Num<KI>::E;
  using EO = typename Num<KO>::E;
  const float inv = 1.f / (float)a.D;
  float w[2 * V] = {};
  if (in) n_load<1, V, CH>(a, q.w, p0, w);
  const long long units = U::count(a, q);
  for (long long unit = (long long)blk * 4 + wave; unit < units; unit += 4LL * q.blocks) {
    const U n(a, q, unit, sc[wave]);
    float sn[V], cs[V];
    n.sines(q, sc[wave], sn, cs);
    const EI* x = (const EI*)q.x + n.b * q.xb + n.t * q.xt;
    EO* y = (EO*)q.y + n.b * q.yb + n.t * q.yt;
    const bool live = in && n.valid;
    // all lanes of a wave run the same number of rounds
    for (int h = n.h0, base = 0; base < n.h1; h += n.step, base += n.step) {
      float u[2 * V] = {};
      const bool on = live && h < n.h1;
      if (on) n_load<KI, V, CH>(a, x + h * q.xh, p0, u);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) ss = fmaf(u[i], u[i], ss);
      const float r = __frsqrt_rn(fmaf(n_sum<LPR>(ss), inv, a.eps));
      float o[2 * V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float ua = u[i] * r * w[i], ub = u[V + i] * r * w[V + i];
        o[i] = ua * cs[i] - ub * sn[i];
        o[V + i] = ub * cs[i] + ua * sn[i];
      }
      if (on) n_store<KO, V, CH>(a, y + h * q.yh, p0, o);
    }
  }
}

// dx, and each block's share of dw.
template <int KI, int KO, int V, int LPR, bool CH>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(const NArgs a) {
  __shared__ float2 sc[4][64 * V];
  using U = Unit<V, LPR>;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % LPR, p0 = c * V;
  int blk;
  const NPart& q = a.p[n_part(a, blk)];
  const bool in = p0 < a.D / 2;
  using EI = typename Num<KI>::E;
  using EO = typename Num<KO>::E;
  const float inv = 1.f / (float)a.D;
  float w[2 * V] = {}, dw[2 * V] = {};
  if (in) n_load<1, V, CH>(a, q.w, p0, w);
  const long long units = U::count(a, q);
  for (long long unit = (long long)blk * 4 + wave; unit < units; unit += 4LL * q.blocks) {
    const U n(a, q, unit, sc[wave]);
    float sn[V], cs[V];
    n.sines(q, sc[wave], sn, cs);
    const EI* x = (const EI*)q.x + n.b * q.xb + n.t * q.xt;
    const EO* dy = (const EO*)q.dy + n.b * q.gb + n.t * q.gt;
    EI* dx = (EI*)q.y + n.b * q.yb + n.t * q.yt;
    const bool live = in && n.valid;
    for (int h = n.h0, base = 0; base < n.h1; h += n.step, base += n.step) {
      float u[2 * V] = {}, d[2 * V] = {};
      const bool on = live && h < n.h1;
      if (on) {
        n_load<KI, V, CH>(a, x + h * q.xh, p0, u);
        n_load<KO, V, CH>(a, dy + h * q.gh, p0, d);
      }
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) ss = fmaf(u[i], u[i], ss);
      const float r = __frsqrt_rn(fmaf(n_sum<LPR>(ss), inv, a.eps));
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float da = d[i] * cs[i] + d[V + i] * sn[i], db = d[V + i] * cs[i] - d[i] * sn[i];
        u[i] = on ? u[i] * r : 0.f;          // eps = 0: no row, no infinity
        u[V + i] = on ? u[V + i] * r : 0.f;
        dw[i] = fmaf(da, u[i], dw[i]);
        dw[V + i] = fmaf(db, u[V + i], dw[V + i]);
        d[i] = da * w[i];
        d[V + i] = db * w[V + i];
        dot = fmaf(d[i], u[i], fmaf(d[V + i], u[V + i], dot));
      }
      dot = n_sum<LPR>(dot) * inv;
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) d[i] = r * (d[i] - u[i] * dot);
      if (on) n_store<KI, V, CH>(a, dx + h * q.yh, p0, d);
    }
  }
  if (!a.part) return;
  __syncthreads();
  float* red = (float*)sc;                            // [4][2 V LPR]
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) {
#pragma unroll
    for (int m = LPR; m < 64; m <<= 1) dw[i] += __shfl_xor(dw[i], m);
    if (lane < LPR) red[wave * (2 * V * LPR) + i * LPR + c] = dw[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * V * LPR; i += 256) {
    const int p = i % LPR * V + i / LPR % V;
    if (p < a.D / 2)
      a.part[(long long)blockIdx.x * a.D + (i / LPR < V ? n_first(a, p) : n_second(a, p))] =
          red[i] + red[2 * V * LPR + i] + red[4 * V * LPR + i] + red[6 * V * LPR + i];
  }
}

// dw of 8 columns of one part: 32 rows of partials at a time, in a fixed order
__global__ __launch_bounds__(256) void qk_norm_rope_dw_kernel(const float* part, int b0, int b1,
                                                              int D, float* dwq, float* dwk) {
  __shared__ float red[32][8];
  const int col = blockIdx.x * 8 + threadIdx.x % 8, r = threadIdx.x / 8;
  const int lo = blockIdx.y ? b0 : 0, hi = blockIdx.y ? b0 + b1 : b0;
  float s = 0.f;
  if (col < D)
    for (int i = lo + r; i < hi; i += 32) s += part[(long long)i * D + col];
  red[r][threadIdx.x % 8] = s;
  __syncthreads();
  if (r == 0 && col < D) {
    s = 0.f;
    for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x % 8];
    float* o = blockIdx.y ? dwk : dwq;
    if (o) o[col] = s;
  }
}

template <int KI, int KO, int V, int LPR, bool CH>
int n_go(const NArgs& a, int grid, bool bwd, hipStream_t st) {
  if (bwd)
    hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<KI, KO, V, LPR, CH>), dim3(grid), dim3(256), 0, st,
                       a);
  else
    hipLaunchKernelGGL((qk_norm_rope_kernel<KI, KO, V, LPR, CH>), dim3(grid), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

// V: pairs per lane of 16-byte chunks
constexpr int n_vec(int type) { return type == 1 ? 4 : 8; }
bool n_chunked(int type, int D, int R, int interleaved) {
  const int v = n_vec(type);
  return interleaved ? D / 2 % v == 0 : R / 2 % v == 0 && (D - R) / 2 % v == 0;
}
// lanes per head
int n_lanes(int type, int D, bool ch) {
  if (!ch) return D <= 64 ? 16 : 64;                // two pairs each
  const int v = n_vec(type), n = (D / 2 + v - 1) / v;
  return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32;
}

template <int KI, int KO>
int n_run(const NArgs& a, int grid, bool bwd, bool ch, int lpr, hipStream_t st) {
  constexpr int V = n_vec(KI);
  if (ch) {
    if (lpr == 4) return n_go<KI, KO, V, 4, true>(a, grid, bwd, st);
    if (lpr == 8) return n_go<KI, KO, V, 8, true>(a, grid, bwd, st);
    if (lpr == 16) return n_go<KI, KO, V, 16, true>(a, grid, bwd, st);
    return n_go<KI, KO, V, 32, true>(a, grid, bwd, st);
  }
  if (lpr == 16) return n_go<KI, KO, 2, 16, false>(a, grid, bwd, st);
  return n_go<KI, KO, 2, 64, false>(a, grid, bwd, st);
}

int n_dispatch(const NArgs& a, int grid, bool bwd, bool ch, int lpr, int ti, int to,
               hipStream_t st) {
  if (ti == 0 && to == 0) return n_run<0, 0>(a, grid, bwd, ch, lpr, st);
  if (ti == 2 && to == 2) return n_run<2, 2>(a, grid, bwd, ch, lpr, st);
  if (ti == 1 && to == 1) return n_run<1, 1>(a, grid, bwd, ch, lpr, st);
  if (ti == 1 && to == 0) return n_run<1, 0>(a, grid, bwd, ch, lpr, st);
  if (ti == 1 && to == 2) return n_run<1, 2>(a, grid, bwd, ch, lpr, st);
  return 1002;
}

// Units of a part (Unit::count)
long long n_units(const NArgs& a, const NPart& p, int lpr) {
  const long long tokens = (long long)p.B * p.T, at_once = 64 / lpr >> p.lg;
  return (tokens + at_once - 1) / at_once * (a.many ? 1 : (p.H + (1 << p.lg) - 1) >> p.lg);
}
// Blocks for both parts, at most `most`, shared by the heads that they have:
// a wave with several units loads its weights once.
void n_blocks(NArgs& a, int lpr, int most) {
  const long long u0 = n_units(a, a.p[0], lpr), u1 = n_units(a, a.p[1], lpr);
  const long long b0 = (u0 + 3) / 4, b1 = (u1 + 3) / 4;
  if (b0 + b1 <= most) {
    a.p[0].blocks = (int)b0;
    a.p[1].blocks = (int)b1;
    return;
  }
  const double r0 = (double)a.p[0].B * a.p[0].T * a.p[0].H;
  const double r1 = (double)a.p[1].B * a.p[1].T * a.p[1].H;
  long long x = (long long)(most * (r0 / (r0 + r1)));
  if (b1 && x > most - 1) x = most - 1;
  if (b0 && x < 1) x = 1;
  if (x > b0) x = b0;
  a.p[0].blocks = (int)x;
  a.p[1].blocks = (int)(most - x < b1 ? most - x : b1);
}

bool n_fill(NArgs& a, const long long* s, const void* q, const void* k, const void* gq,
            const void* gk, void* yq, void* yk, const float* wq, const float* wk, const void* qpos,
            const void* kpos) {
  const void* x[2] = {q, k};
  const void* g[2] = {gq, gk};
  void* y[2] = {yq, yk};
  const float* w[2] = {wq, wk};
  const void* pos[2] = {qpos, kpos};
  for (int i = 0; i < 2; ++i) {
    const long long* t = s + 15 * i;
    NPart& p = a.p[i];
    p = NPart{x[i], t[3], t[4], t[5], g[i], t[6], t[7], t[8], y[i], t[9],
              t[10], t[11], w[i], pos[i], t[12], t[13], t[14], (int)t[0], (int)t[1], (int)t[2], 0, 0};
    for (int j = 0; j < 3; ++j)
      if (t[j] < 0 || t[j] > 1LL << 30) return false;
    if (t[0] * t[1] > 1LL << 30) return false;            // token numbers are 32-bit
    if (!x[i]) p.B = p.T = p.H = 0;
    else if (!y[i] || !w[i]) return false;
  }
  return true;
}

}  // namespace

extern "C" {

int tgfr_qk_norm_rope_ws(int D, long long* floats) {
  if (!floats || D < 2 || D > 256) return 1001;
  *floats = 1024LL * D;
  return 0;
}

static int n_entry(const void* q, const void* k, const void* gq, const void* gk, void* yq,
                   void* yk, const long long* shapes, const float* wq, const float* wk,
                   const void* qpos, const void* kpos, int pos32, const unsigned long long* turn,
                   int R, int axes, int interleaved, int D, float eps, int ti, int to, bool bwd,
                   float* part, float* dwq, float* dwk, void* stream) {
  if (!shapes || D < 2 || D > 256 || D % 2 || R < 0 || R > D || R % 2 || axes < 1 ||
      (R && (!turn || R / 2 % axes)))
    return 1001;
  if (ti < 0 || ti > 2 || to < 0 || to > 2) return 1002;
  NArgs a{};
  if (!n_fill(a, shapes, q, k, gq, gk, yq, yk, wq, wk, qpos, kpos)) return 1001;
  if (bwd && ((q && !gq) || (k && !gk))) return 1001;
  a.turn = turn;
  a.part = part;
  a.D = D;
  a.R = R;
  a.per = R ? R / 2 / axes : 1;
  a.interleaved = interleaved;
  a.pos32 = pos32;
  a.eps = eps;
  const bool ch = n_chunked(ti, D, R, interleaved);
  const int lpr = n_lanes(ti, D, ch);
  long long tokens = 0;
  for (NPart& p : a.p) {
    while ((1 << p.lg) < p.H && (1 << p.lg) < 64 / lpr) ++p.lg;
    tokens += (long long)p.B * p.T;
  }
  // With few tokens the heads of one go to waves of their own, which form its
  // sines again (32 + 8 heads of 128: 512 tokens of both 4.9 us against 5.9, 2048
  // 8.2 against 7.1, 65536 159 against 135).
  a.many = tokens >= 2048;
  const hipStream_t st = (hipStream_t)stream;
  n_blocks(a, lpr, bwd ? 1024 : 4096);
  const int grid = a.p[0].blocks + a.p[1].blocks;
  if (grid)
    if (const int e = n_dispatch(a, grid, bwd, ch, lpr, ti, to, st)) return e;
  if (!part) return 0;
  hipLaunchKernelGGL(qk_norm_rope_dw_kernel, dim3((D + 7) / 8, 2), dim3(256), 0, st, part,
                     a.p[0].blocks, a.p[1].blocks, D, dwq, dwk);
  return (int)hipGetLastError();
}

int tgfr_qk_norm_rope_fwd(const void* q, const void* k, void* yq, void* yk, const long long* shapes,
                          const float* wq, const float* wk, const void* qpos, const void* kpos,
                          int pos32, const unsigned long long* turn, int R, int axes,
                          int interleaved, int D, float eps, int type_in, int type_out,
                          void* stream) {
  return n_entry(q, k, nullptr, nullptr, yq, yk, shapes, wq, wk, qpos, kpos, pos32, turn, R, axes,
                 interleaved, D, eps, type_in, type_out, false, nullptr, nullptr, nullptr, stream);
}

int tgfr_qk_norm_rope_bwd(const void* q, const void* k, const void* dyq, const void* dyk, void* dq,
                          void* dk, const long long* shapes, const float* wq, const float* wk,
                          const void* qpos, const void* kpos, int pos32,
                          const unsigned long long* turn, int R, int axes, int interleaved, int D,
                          float eps, int type_in, int type_out, float* ws, float* dwq, float* dwk,
                          void* stream) {
  return n_entry(q, k, dyq, dyk, dq, dk, shapes, wq, wk, qpos, kpos, pos32, turn, R, axes,
                 interleaved, D, eps, type_in, type_out, true, ws, dwq, dwk, stream);
}

}  // extern "C"
