// fa_rotary.hpp -- rotary position embedding from positions and frequencies.
//
// Pair j (of R / 2) of a row at position p turns by the angle p f_j:
//
//   a' = m (a cos - b sin),  b' = m (b cos + a sin)
//
// with (a, b) the columns (j, R/2 + j) in the half layout and (2j, 2j + 1)
// in the interleaved one; columns R .. D-1 are copied.  The gradient of a
// rotation is the rotation by the negative angle.
//
// Angles are kept in turns, as 64-bit fixed-point fractions: the caller gives
// step_j = f_j / 2 pi mod 1 in units of 2^-64, and p * step_j in wrapping
// integer arithmetic is the fraction of the turn, exact but for the step's
// own rounding (|p| 2^-65 turns: 4e-10 rad at p = 2^31).  An fp32 product
// p * f_j is off by up to 2^-24 p f_j, 0.06 rad at p = 10^6.  The top two bits
// (rounded) are the quadrant, the rest an angle of at most pi/4 for the
// Taylor polynomials of sine and cosine (truncated under 2e-10 in fp32, 5e-17
// and 1e-15 in fp64).
#pragma once

#include "fa_common.hpp"

namespace fa {

struct RotaryTable {
  const int64_t *steps;   // (R / 2)
  double factor;          // m
  int r2;                 // R / 2
  int interleaved;
  int inverse;            // negative angles
};

template <typename F> struct CosSin { F c, s; };

__device__ __forceinline__ void sincos_poly(float x, float &s, float &c) {
  const float z = x * x;
  s = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 +
      z * (-1.0f / 3628800)))));
}

__device__ __forceinline__ void sincos_poly(double x, double &s, double &c) {
  const double z = x * x;
  s = x + x * z * (-1.0 / 6 + z * (1.0 / 120 + z * (-1.0 / 5040 + z * (1.0 / 362880 +
      z * (-1.0 / 39916800 + z * (1.0 / 6227020800.0 + z * (-1.0 / 1307674368000.0)))))));
  c = 1.0 + z * (-0.5 + z * (1.0 / 24 + z * (-1.0 / 720 + z * (1.0 / 40320 +
      z * (-1.0 / 3628800 + z * (1.0 / 479001600.0 + z * (-1.0 / 87178291200.0)))))));
}

// m cos and m sin of position p and a pair's step, in F (fp32 or fp64).
template <typename F>
__device__ __forceinline__ CosSin<F> rotary_cos_sin(int64_t p, int64_t step, F factor) {
  const uint64_t turn = (uint64_t)p * (uint64_t)step;
  const uint64_t quad = (turn + (1ull << 61)) >> 62;
  const int64_t rest = (int64_t)(turn - (quad << 62));   // [-2^61, 2^61): an eighth of a turn
  F x;
  if constexpr (sizeof(F) == 4)
    x = (float)(int32_t)(rest >> 32) * (float)(6.283185307179586 / 4294967296.0);
  else
    x = (double)rest * (6.283185307179586477 / 18446744073709551616.0);
  F s, c;
  sincos_poly(x, s, c);
  const bool odd = quad & 1;
  const F cc = odd ? s : c, ss = odd ? c : s;   // |cos|, |sin| up to sign
  // quadrant 0: (c, s); 1: (-s, c); 2: (-c, -s); 3: (s, -c)
  return CosSin<F>{factor * ((quad == 1 || quad == 2) ? -cc : cc),
                   factor * ((quad & 2) ? -ss : ss)};
}

template <typename E, typename F>
__device__ __forceinline__ void load8(const f16 *p, F *x) {
  const vec8<E> v = *reinterpret_cast<const vec8<E> *>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (F)(float)v[i];
}

// Columns 8c .. 8c+7 of a row, rotated by the row's table cs[R / 2].  The
// partner columns of a half-layout chunk are a load of their own (they come
// from the L1 line that another lane of the wave loads as its own chunk):
// a lane then owns 8 consecutive columns whatever R is, and groups of lanes
// own the 32-column blocks that the 4-bit cache shares a scale over.
// Chunks whose partners are not 8 aligned columns (R % 16) load them one by
// one; the branch is uniform.
template <typename E, typename F>
__device__ __forceinline__ void rotate8(const f16 *row, int c, const CosSin<F> *cs, int r2,
                                        bool interleaved, F *y) {
  F x[8];
  load8<E, F>(row + 8 * c, x);
  if (interleaved) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = 4 * c + j;
      if (p < r2) {
        const CosSin<F> t = cs[p];
        y[2 * j] = x[2 * j] * t.c - x[2 * j + 1] * t.s;
        y[2 * j + 1] = x[2 * j + 1] * t.c + x[2 * j] * t.s;
      } else {
        y[2 * j] = x[2 * j];
        y[2 * j + 1] = x[2 * j + 1];
      }
    }
  } else if ((r2 & 7) == 0) {
    const int d = 8 * c;
    if (d < 2 * r2) {
      const bool low = d < r2;
      F z[8];
      load8<E, F>(row + (low ? d + r2 : d - r2), z);
      const CosSin<F> *t = cs + (low ? d : d - r2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const CosSin<F> v = t[i];
        y[i] = x[i] * v.c + (low ? -z[i] : z[i]) * v.s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = 8 * c + i;
      y[i] = x[i];
      if (d < 2 * r2) {
        const bool low = d < r2;
        const F z = (F)(float)*reinterpret_cast<const E *>(row + (low ? d + r2 : d - r2));
        const CosSin<F> v = cs[low ? d : d - r2];
        y[i] = x[i] * v.c + (low ? -z : z) * v.s;
      }
    }
  }
}

template <typename E>
__device__ __forceinline__ void store8(f16 *p, const float *y) {
  vec8<E> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (E)y[i];
  *reinterpret_cast<vec8<E> *>(p) = v;
}

struct RotaryArgs {
  const f16 *x[2];      // q, k
  f16 *y[2];
  int64_t xs[2][3];     // {b, s, h} strides
  int64_t ys[2][3];
  int heads[2];         // k: 0 where there is none
  RotaryTable rot;
  const void *positions;
  int64_t pb, ps;       // strides of positions
  int pos64;            // int64 positions
  int S, D;
  int64_t tokens;       // B * S
};

// One workgroup rotates every head of TOK tokens (or, split over gridDim.y,
// part of them).  Bound by HBM: each element is read and written once.  The
// cosines and sines of a token are shared by its heads: computed once per
// workgroup into LDS, then read by one lane per 8 columns.
constexpr int kRotaryThreads = 256;

__device__ __forceinline__ int64_t rotary_position(const void *positions, int pos64, int64_t i) {
  return pos64 ? static_cast<const int64_t *>(positions)[i]
               : (int64_t) static_cast<const int32_t *>(positions)[i];
}

template <typename E, int TOK>
__global__ __launch_bounds__(kRotaryThreads) void fa_rotary_kernel(RotaryArgs a) {
  extern __shared__ char smem[];
  CosSin<float> *cs = reinterpret_cast<CosSin<float> *>(smem);   // [TOK][R / 2]
  const int r2 = a.rot.r2;
  const int64_t n0 = (int64_t)blockIdx.x * TOK;
  const int nt = (int)min((int64_t)TOK, a.tokens - n0);
  for (int i = threadIdx.x; i < nt * r2; i += kRotaryThreads) {
    const int t = i / r2, j = i - t * r2;
    const uint32_t n = (uint32_t)(n0 + t), b = n / (uint32_t)a.S, s = n - b * (uint32_t)a.S;
    const int64_t p = rotary_position(a.positions, a.pos64, b * a.pb + s * a.ps);
    CosSin<float> v = rotary_cos_sin<float>(p, a.rot.steps[j], (float)a.rot.factor);
    if (a.rot.inverse) v.s = -v.s;
    cs[i] = v;
  }
  __syncthreads();
  const int chunks = a.D / 8, heads = a.heads[0] + a.heads[1];
  const int work = nt * heads * chunks;
  for (int i = blockIdx.y * kRotaryThreads + threadIdx.x; i < work;
       i += gridDim.y * kRotaryThreads) {
    const int c = i % chunks, th = i / chunks, t = th / heads, hh = th - t * heads;
    const int side = hh >= a.heads[0];
    const int h = side ? hh - a.heads[0] : hh;
    const uint32_t n = (uint32_t)(n0 + t), b = n / (uint32_t)a.S, s = n - b * (uint32_t)a.S;
    const f16 *row = a.x[side] + b * a.xs[side][0] + s * a.xs[side][1] + h * a.xs[side][2];
    f16 *out = a.y[side] + b * a.ys[side][0] + s * a.ys[side][1] + h * a.ys[side][2];
    float y[8];
    rotate8<E, float>(row, c, cs + t * r2, r2, a.rot.interleaved != 0, y);
    store8<E>(out + 8 * c, y);
  }
}

}  // namespace fa
