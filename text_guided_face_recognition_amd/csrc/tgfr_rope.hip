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
// Bound by memory: x is read once and y written once.  16 bytes per lane and
// load; a wave takes one token, LPR lanes per head, so the sines of a lane's
// pairs are formed once and serve all heads of the token.
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
  int blocks;           // backward: blocks of this part
};
struct NArgs {
  NPart p[2];
  const unsigned long long* turn;   // [R / 2]
  float* part;          // backward: [blocks][D] partial dw
  int D, R, per, interleaved, pos32, heads;   // heads: per wave and unit
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
struct Place {
  int p0;        // first pair; pairs past D / 2 do not exist
  int a0, b0;
};
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

// sines of a lane's pairs at one token
template <int V>
__device__ __forceinline__ void n_angles(const NArgs& a, const NPart& q, int b, int t, int p0,
                                         const unsigned long long (&turn)[V], float (&cs)[V],
                                         float (&sn)[V]) {
  long long last = 0;
  int axis = -1;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (p0 + i < a.R / 2) {
      const int ax = (p0 + i) / a.per;
      if (ax != axis) {
        axis = ax;
        last = t;
        if (q.pos) {
          const long long at = b * q.pb + t * q.pt + ax * q.pa;
          last = a.pos32 ? ((const int*)q.pos)[at] : ((const long long*)q.pos)[at];
        }
      }
      const unsigned long long f = (unsigned long long)last * turn[i];
      // signed fraction of a turn, [-1/2, 1/2)
      const float turns = fmaf((float)(uint32_t)f, 0x1p-64f, (float)(int32_t)(f >> 32) * 0x1p-32f);
      sincospif(2.f * turns, &sn[i], &cs[i]);
    }
  }
}

template <int LPR>
__device__ __forceinline__ float n_sum(float v) {
#pragma unroll
  for (int m = LPR / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// One unit of a wave: a token and `heads` of its heads, IT times 64 / LPR at
// once.
template <int KI, int KO, int V, int LPR, bool CH>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const NArgs a) {
  const int lane = threadIdx.x % 64, c = lane % LPR, g = lane / LPR;
  constexpr int HPW = 64 / LPR;
  long long unit = (long long)blockIdx.x * 4 + threadIdx.x / 64;
  int k = 0;
  const long long n0 = (long long)a.p[0].B * a.p[0].T * ((a.p[0].H + a.heads - 1) / a.heads);
  if (unit >= n0) {
    unit -= n0;
    k = 1;
  }
  const NPart& q = a.p[k];
  const int hu = (q.H + a.heads - 1) / a.heads;
  if (unit >= (long long)q.B * q.T * hu) return;
  const long long tok = unit / hu;
  const int b = (int)(tok / q.T), t = (int)(tok % q.T);
  const int h0 = (int)(unit % hu) * a.heads, h1 = min(q.H, h0 + a.heads);
  const int p0 = c * V;
  const bool in = p0 < a.D / 2;
  using EI = typename Num<KI>::E;
  using EO = typename Num<KO>::E;

  unsigned long long turn[V];
  float w[2 * V], cs[V], sn[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    turn[i] = p0 + i < a.R / 2 ? a.turn[p0 + i] : 0;
    const bool e = p0 + i < a.D / 2;
    w[i] = e ? q.w[n_first(a, p0 + i)] : 0.f;
    w[V + i] = e ? q.w[n_second(a, p0 + i)] : 0.f;
  }
  n_angles<V>(a, q, b, t, p0, turn, cs, sn);
  const EI* x = (const EI*)q.x + b * q.xb + t * q.xt;
  EO* y = (EO*)q.y + b * q.yb + t * q.yt;
  for (int h = h0 + g; h < h1; h += HPW) {
    float u[2 * V] = {};
    if (in) n_load<KI, V, CH>(a, x + h * q.xh, p0, u);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) ss = fmaf(u[i], u[i], ss);
    const float r = __frsqrt_rn(n_sum<LPR>(ss) / (float)a.D + a.eps);
    float o[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float ua = u[i] * r * w[i], ub = u[V + i] * r * w[V + i];
      o[i] = ua * cs[i] - ub * sn[i];
      o[V + i] = ub * cs[i] + ua * sn[i];
    }
    if (in) n_store<KO, V, CH>(a, y + h * q.yh, p0, o);
  }
}

// dx, and each block's share of dw.
template <int KI, int KO, int V, int LPR, bool CH>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(const NArgs a) {
  constexpr int HPW = 64 / LPR;
  __shared__ float red[4][2 * 64 * V];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % LPR, g = lane / LPR;
  const int k = (int)blockIdx.x >= a.p[0].blocks;
  const NPart& q = a.p[k];
  const int blk = k ? blockIdx.x - a.p[0].blocks : blockIdx.x;
  const int hu = (q.H + a.heads - 1) / a.heads;
  const long long units = (long long)q.B * q.T * hu;
  const int p0 = c * V;
  const bool in = p0 < a.D / 2;
  using EI = typename Num<KI>::E;
  using EO = typename Num<KO>::E;

  unsigned long long turn[V];
  float w[2 * V], cs[V], sn[V], dw[2 * V] = {};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    turn[i] = p0 + i < a.R / 2 ? a.turn[p0 + i] : 0;
    const bool e = p0 + i < a.D / 2;
    w[i] = e ? q.w[n_first(a, p0 + i)] : 0.f;
    w[V + i] = e ? q.w[n_second(a, p0 + i)] : 0.f;
  }
  for (long long unit = (long long)blk * 4 + wave; unit < units; unit += 4LL * q.blocks) {
    const long long tok = unit / hu;
    const int b = (int)(tok / q.T), t = (int)(tok % q.T);
    const int h0 = (int)(unit % hu) * a.heads, h1 = min(q.H, h0 + a.heads);
    n_angles<V>(a, q, b, t, p0, turn, cs, sn);
    const EI* x = (const EI*)q.x + b * q.xb + t * q.xt;
    const EO* dy = (const EO*)q.dy + b * q.gb + t * q.gt;
    EI* dx = (EI*)q.y + b * q.yb + t * q.yt;
    for (int h = h0 + g; h < h1; h += HPW) {
      float u[2 * V] = {}, d[2 * V] = {};
      if (in) {
        n_load<KI, V, CH>(a, x + h * q.xh, p0, u);
        n_load<KO, V, CH>(a, dy + h * q.gh, p0, d);
      }
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) ss = fmaf(u[i], u[i], ss);
      const float r = __frsqrt_rn(n_sum<LPR>(ss) / (float)a.D + a.eps);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float da = d[i] * cs[i] + d[V + i] * sn[i], db = d[V + i] * cs[i] - d[i] * sn[i];
        u[i] *= r;
        u[V + i] *= r;
        dw[i] = fmaf(da, u[i], dw[i]);
        dw[V + i] = fmaf(db, u[V + i], dw[V + i]);
        d[i] = da * w[i];
        d[V + i] = db * w[V + i];
        dot = fmaf(d[i], u[i], fmaf(d[V + i], u[V + i], dot));
      }
      dot = n_sum<LPR>(dot) / (float)a.D;
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) d[i] = r * (d[i] - u[i] * dot);
      if (in) n_store<KI, V, CH>(a, dx + h * q.yh, p0, d);
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) {
#pragma unroll
    for (int m = LPR; m < 64; m <<= 1) dw[i] += __shfl_xor(dw[i], m);
    if (g == 0) red[wave][i * LPR + c] = dw[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * V * LPR; i += 256) {
    const int p = i % LPR * V + i / LPR % V;
    if (p < a.D / 2)
      a.part[(long long)blockIdx.x * a.D + (i / LPR < V ? n_first(a, p) : n_second(a, p))] =
          red[0][i] + red[1][i] + red[2][i] + red[3][i];
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
int n_lanes(int type, int D, bool ch) {
  const int v = ch ? n_vec(type) : 2, n = (D / 2 + v - 1) / v;
  return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 64;
}

template <int KI, int KO>
int n_run(const NArgs& a, int grid, bool bwd, bool ch, int lpr, hipStream_t st) {
  constexpr int V = n_vec(KI);
  if (ch) {
    if (lpr == 8) return n_go<KI, KO, V, 8, true>(a, grid, bwd, st);
    if (lpr == 16) return n_go<KI, KO, V, 16, true>(a, grid, bwd, st);
    return n_go<KI, KO, V, 32, true>(a, grid, bwd, st);
  }
  if (lpr <= 16) return n_go<KI, KO, 2, 16, false>(a, grid, bwd, st);
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

// heads per unit: a whole token per wave shares its sines among the heads;
// with few tokens the heads go to waves of their own
int n_heads(long long tokens, int H, int lpr) {
  const int at_once = 64 / lpr;
  return tokens >= 8192 ? (H + at_once - 1) / at_once * at_once : at_once;
}
long long n_units(const NPart& p, int heads) {
  return (long long)p.B * p.T * ((p.H + heads - 1) / heads);
}
// blocks of the backward for both parts (at most 1024 in all, shared by size)
void n_blocks(NArgs& a) {
  const long long u0 = n_units(a.p[0], a.heads), u1 = n_units(a.p[1], a.heads);
  const long long b0 = (u0 + 3) / 4, b1 = (u1 + 3) / 4, all = b0 + b1;
  if (all <= 1024) {
    a.p[0].blocks = (int)b0;
    a.p[1].blocks = (int)b1;
  } else {
    long long x = 1024 * b0 / all;
    if (x < 1 && b0) x = 1;
    if (x > 1023 && b1) x = 1023;
    a.p[0].blocks = (int)x;
    a.p[1].blocks = (int)(1024 - x);
  }
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
              t[10], t[11], w[i], pos[i], t[12], t[13], t[14], (int)t[0], (int)t[1], (int)t[2], 0};
    for (int j = 0; j < 3; ++j)
      if (t[j] < 0 || t[j] > 0x7fffffffLL) return false;
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
  int lpr = n_lanes(ti, D, ch);
  if (!ch) lpr = lpr <= 16 ? 16 : 64;
  const long long tokens =
      (long long)a.p[0].B * a.p[0].T + (long long)a.p[1].B * a.p[1].T;
  const int H = a.p[0].H > a.p[1].H ? a.p[0].H : a.p[1].H;
  a.heads = n_heads(tokens, H < 1 ? 1 : H, lpr);
  const long long units = n_units(a.p[0], a.heads) + n_units(a.p[1], a.heads);
  if (units > 0x1ffffffffLL) return 1001;
  const hipStream_t st = (hipStream_t)stream;
  if (!bwd) {
    if (!units) return 0;
    return n_dispatch(a, (int)((units + 3) / 4), false, ch, lpr, ti, to, st);
  }
  n_blocks(a);
  const int grid = a.p[0].blocks + a.p[1].blocks;
  if (grid)
    if (const int e = n_dispatch(a, grid, true, ch, lpr, ti, to, st)) return e;
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
