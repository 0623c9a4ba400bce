// C entries of cross attention (kernels: tgfr_xattn.h, one file per type).
#include <algorithm>

#include "tgfr_xattn.h"

using namespace tgfr;

namespace {

int x_dispatch(const XArgs& a, int type, int what, void* stream) {
  return type == 0   ? xattn_run_bf16(a, what, stream)
         : type == 1 ? xattn_run_f32(a, what, stream)
                     : xattn_run_f16(a, what, stream);
}

int x_shape(XArgs& a, int type, int B, int Tq, int Tk, int H, int Hk, int D) {
  if (type < 0 || type > 2) return 1002;
  if (B < 1 || Tq < 1 || Tk < 1 || H < 1 || Hk < 1 || H % Hk || D < 1 || D > 256) return 1001;
  // row and state numbers, and the grids (one block or wave per row), are 32-bit
  const long long rows = (long long)Tq * (H / Hk), lim = 1LL << 30;
  if (H / Hk > 32768 || rows > lim || Tk > lim || rows * B * Hk > lim ||
      (long long)Tk * B * Hk > lim || (long long)B * Hk * 256 > X_THREADS)
    return 1001;
  a.B = B;
  a.Tq = Tq;
  a.Tk = Tk;
  a.H = H;
  a.Hk = Hk;
  a.G = H / Hk;
  a.D = D;
  a.R = (int)rows;
  a.per_g = a.G == 1 ? 0 : (uint32_t)(((1ULL << 32) + a.G - 1) / a.G);
  return 0;
}

const uint8_t* const ANY_MASK = (const uint8_t*)1;    // (for the plan, never read)

long long x_part(const XArgs& a, int type, int what) {
  const bool kv = what == X_DKV;
  const XPlan p = x_plan(a, type, what);
  if (p.splits == 1) return 0;
  const long long n = (long long)p.splits * a.B * a.Hk * (kv ? a.Tk : a.R);
  return n * a.D * (kv ? 2 : 1) + (what == X_FWD ? 2 * n : 0);
}

// The kernels read tiles of up to 128 rows by 32-bit offsets from the first.
bool x_span(const XArgs& a, const XView& v, int type, int heads) {
  const long long es = type == 1 ? 4 : 2;
  return v.st >= 0 && v.sh >= 0 && (160 * v.st + heads * v.sh + 256) * es < 1LL << 31;
}
// Whole chunks of 16 bytes at 4-byte alignment.
bool x_chunks(const XArgs& a, const XView& v) {
  return a.D % 8 == 0 && !((uintptr_t)v.p & 3) && !((v.sb | v.st | v.sh) & 1);
}
int x_reading(XArgs& a, int type) {
  if (!x_span(a, a.q, type, a.G) || !x_span(a, a.k, type, 1) || !x_span(a, a.v, type, 1) ||
      (a.dout.p && !x_span(a, a.dout, type, a.G)))
    return 1001;
  a.fast_k = x_chunks(a, a.k) && x_chunks(a, a.v);
  a.fast_q = x_chunks(a, a.q) && x_chunks(a, a.dout) && 32 % a.G == 0;
  return 0;
}

XView view(const void* p, const long long* s) { return XView{(void*)p, s[0], s[1], s[2]}; }

}  // namespace

extern "C" {

int tgfr_cross_attention_ws(int B, int Tq, int Tk, int H, int Hk, int D, int type, int backward,
                            long long* floats) {
  XArgs a{};
  if (!floats) return 1001;
  if (const int e = x_shape(a, type, B, Tq, Tk, H, Hk, D)) return e;
  // enough with a mask and without
  long long n = 0;
  for (const uint8_t* mask : {(const uint8_t*)nullptr, ANY_MASK}) {
    a.mask = mask;
    if (!backward)
      n = std::max(n, x_part(a, type, X_FWD));
    else
      n = std::max({n, x_part(a, type, X_DQ), x_part(a, type, X_DKV)});
  }
  if (backward)
    n += (long long)B * Hk * (type == 2 ? 2LL * a.R + x_chunks_of_v(a) : a.R);
  *floats = n;
  return 0;
}

int tgfr_cross_attention_fwd(const void* q, const void* k, const void* v, void* o,
                             const long long* strides, const int* q_lens, const int* kv_lens,
                             const uint8_t* mask, long long mask_sb, int B, int Tq, int Tk, int H,
                             int Hk, int D, float scale, int type, float* lse, float* ws,
                             void* stream) {
  XArgs a{};
  if (const int e = x_shape(a, type, B, Tq, Tk, H, Hk, D)) return e;
  if (!q || !k || !v || !o || !strides || !(scale > 0.f)) return 1001;
  a.mask = mask;
  const long long n = x_part(a, type, X_FWD);
  if (n && !ws) return 1001;
  a.q = view(q, strides);
  a.k = view(k, strides + 3);
  a.v = view(v, strides + 6);
  a.o = view(o, strides + 9);
  if (const int e = x_reading(a, type)) return e;
  a.q_lens = q_lens;
  a.kv_lens = kv_lens;
  a.mask_sb = mask_sb;
  a.scale = scale;
  a.lse = lse;
  if (n) {
    a.part_ml = ws;
    a.part = ws + 2 * (n / (D + 2));
  }
  return x_dispatch(a, type, X_FWD, stream);
}

int tgfr_cross_attention_bwd(const void* q, const void* k, const void* v, const void* o,
                             const void* dout, void* dq, void* dk, void* dv,
                             const long long* strides, const int* q_lens, const int* kv_lens,
                             const uint8_t* mask, long long mask_sb, int B, int Tq, int Tk, int H,
                             int Hk, int D, float scale, int type, const float* lse, float* ws,
                             void* stream) {
  XArgs a{};
  if (const int e = x_shape(a, type, B, Tq, Tk, H, Hk, D)) return e;
  if (!q || !k || !v || !o || !dout || !dq || (dk == nullptr) != (dv == nullptr) || !strides ||
      !lse || !ws || !(scale > 0.f))
    return 1001;
  a.q = view(q, strides);
  a.k = view(k, strides + 3);
  a.v = view(v, strides + 6);
  a.o = view(o, strides + 9);
  a.dout = view(dout, strides + 12);
  a.dq = view(dq, strides + 15);
  if (const int e = x_reading(a, type)) return e;
  a.q_lens = q_lens;
  a.kv_lens = kv_lens;
  a.mask = mask;
  a.mask_sb = mask_sb;
  a.scale = scale;
  a.lse = (float*)lse;
  a.delta = ws;
  a.part = ws + (long long)B * Hk * a.R;
  if (type == 2) {
    a.chunks = x_chunks_of_v(a);
    a.size = a.part;
    a.vmax = a.size + (long long)B * Hk * a.R;
    a.part = a.vmax + (long long)B * Hk * a.chunks;
  }
  if (const int e = x_dispatch(a, type, X_DQ, stream)) return e;
  if (!dk) return 0;
  a.dk = view(dk, strides + 18);
  a.dv = view(dv, strides + 21);
  return x_dispatch(a, type, X_DKV, stream);
}

}  // extern "C"
