// Rotary positions with several axes (tdx_rotary_axes).
//
// One pass over x: 2 N bytes of the type, bound by HBM.  The angle pos * base^(-i/n) does not depend on the head, so a workgroup takes
// the angles of its TB tokens once (LDS, one {cos, sin} per token and pair) and applies them to all heads with 16-byte loads and stores.
// An angle is formed as a number of turns in 64 bits (the rates are divided by 2 pi on the host) and its whole turns are dropped before
// it is rounded to 32: at position 1e6 a 32-bit product alone is off by 0.06.
// Measured: 336 MB of bf16 read and written in 66 us (5.1 TB/s; a copy reaches 5.2).
#include "tdx_common.h"

#include <cmath>

namespace {

constexpr int kMaxPairs = 128;

struct RotArgs {
  const void* x;
  void* out;
  const float* pos;
  long x_bs, x_ts, x_hs, o_bs, o_ts, o_hs, p_bs, p_ts, p_as;
  int T, H, D, pairs, tb;
  long tokens;
  float sign;
  double rate[kMaxPairs];           // turns per unit of position
  unsigned char axis[kMaxPairs];
};

template <typename T, int LAYOUT, bool VECTOR>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs a) {
  constexpr int VEC = Elem<T>::kVec;
  extern __shared__ float2 turn[];   // [tb][pairs] {cos, sin}
  const long tok0 = (long)blockIdx.x * a.tb;
  const int ntok = (int)min((long)a.tb, a.tokens - tok0);
  for (int i = threadIdx.x; i < ntok * a.pairs; i += 256) {
    const int tl = i / a.pairs, m = i - tl * a.pairs;
    const long tok = tok0 + tl;
    const long b = tok / a.T, t = tok - b * a.T;
    const double rev = (double)a.pos[b * a.p_bs + t * a.p_ts + a.axis[m] * a.p_as] * a.rate[m];
    const float r = (float)(rev - __builtin_rint(rev));
    float s, c;
    sincospif(2.0f * r, &s, &c);
    turn[i] = make_float2(c, a.sign * s);
  }
  __syncthreads();
  const int P = a.pairs;
  if constexpr (VECTOR) {
    // an item is one vector of the row (pairs layout) or two that are turned against each other (halves), or one vector to copy
    const int nrot = LAYOUT == TDX_ROTARY_HALVES ? P / VEC : 2 * P / VEC;
    const int nv = nrot + (a.D - 2 * P) / VEC;
    const int per_tok = a.H * nv;
    for (int i = threadIdx.x; i < ntok * per_tok; i += 256) {
      const int tl = i / per_tok, hv = i - tl * per_tok;
      const int h = hv / nv, v = hv - h * nv;
      const long tok = tok0 + tl;
      const long b = tok / a.T, t = tok - b * a.T;
      const T* xr = (const T*)a.x + b * a.x_bs + t * a.x_ts + h * a.x_hs;
      T* yr = (T*)a.out + b * a.o_bs + t * a.o_ts + h * a.o_hs;
      const float2* tr = turn + tl * P;
      if (v >= nrot) {
        const int d = 2 * P + (v - nrot) * VEC;
        *reinterpret_cast<u32x4*>(yr + d) = *reinterpret_cast<const u32x4*>(xr + d);
      } else if constexpr (LAYOUT == TDX_ROTARY_HALVES) {
        const int m = v * VEC;
        float x0[VEC], x1[VEC], y0[VEC], y1[VEC];
        Elem<T>::unpack(*reinterpret_cast<const u32x4*>(xr + m), x0);
        Elem<T>::unpack(*reinterpret_cast<const u32x4*>(xr + P + m), x1);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 cs = tr[m + j];
          y0[j] = x0[j] * cs.x - x1[j] * cs.y;
          y1[j] = x0[j] * cs.y + x1[j] * cs.x;
        }
        *reinterpret_cast<u32x4*>(yr + m) = Elem<T>::pack(y0);
        *reinterpret_cast<u32x4*>(yr + P + m) = Elem<T>::pack(y1);
      } else {
        const int m = v * (VEC / 2);
        float x0[VEC], y0[VEC];
        Elem<T>::unpack(*reinterpret_cast<const u32x4*>(xr + 2 * m), x0);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const float2 cs = tr[m + j];
          y0[2 * j] = x0[2 * j] * cs.x - x0[2 * j + 1] * cs.y;
          y0[2 * j + 1] = x0[2 * j] * cs.y + x0[2 * j + 1] * cs.x;
        }
        *reinterpret_cast<u32x4*>(yr + 2 * m) = Elem<T>::pack(y0);
      }
    }
  } else {
    const int nv = P + (a.D - 2 * P);   // pairs, then channels to copy
    const int per_tok = a.H * nv;
    for (int i = threadIdx.x; i < ntok * per_tok; i += 256) {
      const int tl = i / per_tok, hv = i - tl * per_tok;
      const int h = hv / nv, m = hv - h * nv;
      const long tok = tok0 + tl;
      const long b = tok / a.T, t = tok - b * a.T;
      const T* xr = (const T*)a.x + b * a.x_bs + t * a.x_ts + h * a.x_hs;
      T* yr = (T*)a.out + b * a.o_bs + t * a.o_ts + h * a.o_hs;
      if (m >= P) {
        yr[P + m] = xr[P + m];
        continue;
      }
      const int d0 = LAYOUT == TDX_ROTARY_HALVES ? m : 2 * m, d1 = LAYOUT == TDX_ROTARY_HALVES ? m + P : 2 * m + 1;
      const float2 cs = turn[tl * P + m];
      const float x0 = Elem<T>::ld(xr + d0), x1 = Elem<T>::ld(xr + d1);
      yr[d0] = (T)(x0 * cs.x - x1 * cs.y);
      yr[d1] = (T)(x0 * cs.y + x1 * cs.x);
    }
  }
}

template <typename T, int LAYOUT>
void launch(const RotArgs& a, bool vec, hipStream_t st) {
  const dim3 grid((unsigned)((a.tokens + a.tb - 1) / a.tb));
  const size_t lds = (size_t)a.tb * a.pairs * sizeof(float2);
  if (vec) hipLaunchKernelGGL((rotary_kernel<T, LAYOUT, true>), grid, dim3(256), lds, st, a);
  else hipLaunchKernelGGL((rotary_kernel<T, LAYOUT, false>), grid, dim3(256), lds, st, a);
}

}  // namespace

extern "C" int tdx_rotary_axes(const tdx_rotary_desc* d, void* stream) {
  TDX_CHECK_ARG(d, "tdx_rotary_axes: null descriptor");
  TDX_CHECK_ARG(d->dtype == TDX_F32 || d->dtype == TDX_BF16, "tdx_rotary_axes: bad dtype %d", d->dtype);
  TDX_CHECK_ARG(d->layout == TDX_ROTARY_HALVES || d->layout == TDX_ROTARY_PAIRS, "tdx_rotary_axes: bad layout %d", d->layout);
  TDX_CHECK_ARG(d->B >= 0 && d->T >= 0 && d->H >= 0 && d->D >= 1 && d->D <= 256, "tdx_rotary_axes: bad shape B=%d T=%d H=%d D=%d (D 1..256)", d->B, d->T, d->H, d->D);
  TDX_CHECK_ARG(d->H <= 65536, "tdx_rotary_axes: H=%d (at most 65536)", d->H);
  TDX_CHECK_ARG(d->naxes >= 1 && d->naxes <= 8, "tdx_rotary_axes: %d axes (1..8)", d->naxes);
  RotArgs a;
  a.pairs = 0;
  for (int ax = 0; ax < d->naxes; ++ax) {
    TDX_CHECK_ARG(d->sections[ax] >= 0 && d->sections[ax] <= kMaxPairs - a.pairs && std::isfinite(d->base[ax]) && d->base[ax] > 0.0,
                  "tdx_rotary_axes: axis %d: %d pairs, base %g", ax, d->sections[ax], d->base[ax]);
    for (int i = 0; i < d->sections[ax]; ++i) {
      a.rate[a.pairs + i] = std::pow(d->base[ax], -(double)i / d->sections[ax]) * 0.15915494309189533577;   // 1 / (2 pi)
      a.axis[a.pairs + i] = (unsigned char)ax;
    }
    a.pairs += d->sections[ax];
  }
  TDX_CHECK_ARG(a.pairs >= 1 && 2 * a.pairs <= d->D, "tdx_rotary_axes: the sections hold %d pairs, a head has %d channels", a.pairs, d->D);
  if (d->B == 0 || d->T == 0 || d->H == 0) return TDX_OK;
  TDX_CHECK_ARG(d->x && d->out && d->pos, "tdx_rotary_axes: null pointer");
  TDX_CHECK_ARG(d->x != d->out || (d->x_bs == d->out_bs && d->x_ts == d->out_ts && d->x_hs == d->out_hs), "tdx_rotary_axes: in place needs equal strides");
  a.x = d->x, a.out = d->out, a.pos = d->pos;
  a.x_bs = d->x_bs, a.x_ts = d->x_ts, a.x_hs = d->x_hs, a.o_bs = d->out_bs, a.o_ts = d->out_ts, a.o_hs = d->out_hs;
  a.p_bs = d->pos_bs, a.p_ts = d->pos_ts, a.p_as = d->pos_as;
  a.T = d->T, a.H = d->H, a.D = d->D, a.tokens = (long)d->B * d->T, a.sign = d->inverse ? -1.0f : 1.0f;
  // tokens per workgroup: 8 when that still leaves four workgroups a CU, fewer for short calls
  a.tb = 8;
  while (a.tb > 1 && a.tokens < (long)a.tb * 1024) a.tb >>= 1;
  TDX_CHECK_ARG((a.tokens + a.tb - 1) / a.tb * 256 <= 0xffffffffL, "tdx_rotary_axes: too many tokens");
  const int vec = d->dtype == TDX_F32 ? 4 : 8;
  const long str = a.x_bs | a.x_ts | a.x_hs | a.o_bs | a.o_ts | a.o_hs;
  const bool v = (((uintptr_t)a.x | (uintptr_t)a.out) & 15) == 0 && str % vec == 0 && d->D % vec == 0 &&
                 (d->layout == TDX_ROTARY_HALVES ? a.pairs % vec == 0 : (2 * a.pairs) % vec == 0);
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == TDX_F32) {
    if (d->layout == TDX_ROTARY_HALVES) launch<float, TDX_ROTARY_HALVES>(a, v, st);
    else launch<float, TDX_ROTARY_PAIRS>(a, v, st);
  } else {
    if (d->layout == TDX_ROTARY_HALVES) launch<__bf16, TDX_ROTARY_HALVES>(a, v, st);
    else launch<__bf16, TDX_ROTARY_PAIRS>(a, v, st);
  }
  TDX_CHECK_LAUNCH("rotary_kernel");
  return TDX_OK;
}
