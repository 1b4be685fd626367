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

// Place of pair j in a row's table of cosines and sines in LDS: lanes that own
// consecutive chunks of 8 columns read consecutive entries.
__device__ __forceinline__ int pair_slot(int j, int r2) { return (j & 7) * ((r2 + 7) >> 3) + (j >> 3); }
// Entries of a row's table.
__host__ __device__ __forceinline__ int pair_slots(int r2) { return 8 * ((r2 + 7) >> 3); }

// Columns 8c .. 8c+7 of a row, rotated by the row's table cs.  The partner
// columns of a half-layout chunk are a load of their own (they come from the L1
// line that another lane of the wave loads as its own chunk): a lane then owns 8
// consecutive columns whatever R is, and groups of 4 lanes own the 32-column
// blocks that the 4-bit cache shares a scale over.  Chunks whose partners
// are not 8 aligned columns (R % 16) load them one by one; the branch is uniform.
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
        const CosSin<F> t = cs[pair_slot(p, r2)];
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
      const CosSin<F> *t = cs + ((low ? d : d - r2) >> 3);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const CosSin<F> v = t[i * (r2 >> 3)];
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
        const CosSin<F> v = cs[pair_slot(low ? d : d - r2, r2)];
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

// Units of a row, one lane's work each: in the half layout with R % 16 = 0 two
// chunks of 8 columns that are each other's partners (each is loaded, and its
// cosines read, once) or one behind R; else one chunk.
__host__ __device__ __forceinline__ int rotary_units(int r2, bool interleaved, int D) {
  return !interleaved && (r2 & 7) == 0 ? D / 8 - r2 / 8 : D / 8;
}

template <typename E>
__device__ __forceinline__ void rotate_unit(const f16 *row, f16 *out, int u,
                                            const CosSin<float> *cs, int r2, bool interleaved) {
  const int pairs = r2 >> 3;
  if (!interleaved && (r2 & 7) == 0) {
    if (u < pairs) {
      float x[8], z[8], y[8];
      load8<E, float>(row + 8 * u, x);
      load8<E, float>(row + 8 * u + r2, z);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const CosSin<float> v = cs[u + i * pairs];
        y[i] = x[i] * v.c - z[i] * v.s;
        z[i] = z[i] * v.c + x[i] * v.s;
      }
      store8<E>(out + 8 * u, y);
      store8<E>(out + 8 * u + r2, z);
    } else {
      const int d = 8 * (u + pairs);
      *reinterpret_cast<u32x4 *>(out + d) = *reinterpret_cast<const u32x4 *>(row + d);
    }
  } else {
    float y[8];
    rotate8<E, float>(row, u, cs, r2, interleaved, y);
    store8<E>(out + 8 * u, y);
  }
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
  int S, units, unit_shift;   // units of a row, and log2 of the lanes for them
  int64_t tokens;       // B * S
};

// One workgroup rotates every head of TOK tokens (or, split over gridDim.y,
// part of them).  Bound by HBM: each element is read and written once.  The
// cosines and sines of a token are shared by its heads: computed once per
// workgroup into LDS, then read by one lane per unit.  Lanes keep their unit and
// walk the (token, head) rows, so that the sweep has no division.
constexpr int kRotaryThreads = 256;

__device__ __forceinline__ int64_t rotary_position(const void *positions, int pos64, int64_t i) {
  return pos64 ? static_cast<const int64_t *>(positions)[i]
               : (int64_t) static_cast<const int32_t *>(positions)[i];
}

template <typename E, int TOK>
__global__ __launch_bounds__(kRotaryThreads) void fa_rotary_kernel(RotaryArgs a) {
  extern __shared__ char smem[];
  CosSin<float> *cs = reinterpret_cast<CosSin<float> *>(smem);   // [TOK][pair_slots]
  __shared__ int64_t s_x[TOK][2], s_y[TOK][2];                   // a token's row offsets
  const int r2 = a.rot.r2, slots = pair_slots(r2), tid = threadIdx.x;
  const int64_t n0 = (int64_t)blockIdx.x * TOK;
  const int nt = (int)min((int64_t)TOK, a.tokens - n0);
  if (tid < nt) {
    const uint32_t n = (uint32_t)(n0 + tid), b = n / (uint32_t)a.S, s = n - b * (uint32_t)a.S;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s_x[tid][i] = b * a.xs[i][0] + s * a.xs[i][1];
      s_y[tid][i] = b * a.ys[i][0] + s * a.ys[i][1];
    }
  }
  for (int i = tid; i < nt * r2; i += kRotaryThreads) {
    const int t = i / r2, j = i - t * r2;
    const uint32_t n = (uint32_t)(n0 + t), b = n / (uint32_t)a.S, s = n - b * (uint32_t)a.S;
    const int64_t p = rotary_position(a.positions, a.pos64, b * a.pb + s * a.ps);
    CosSin<float> v = rotary_cos_sin<float>(p, a.rot.steps[j], (float)a.rot.factor);
    if (a.rot.inverse) v.s = -v.s;
    cs[t * slots + pair_slot(j, r2)] = v;
  }
  __syncthreads();
  const int u = tid & ((1 << a.unit_shift) - 1), lanes = kRotaryThreads >> a.unit_shift;
  if (u >= a.units) return;
  const int heads = a.heads[0] + a.heads[1], step = lanes * gridDim.y;
  const int dt = step / heads, dh = step - dt * heads;
  int t = (blockIdx.y * lanes + (tid >> a.unit_shift)), hh = t % heads;
  t /= heads;
  for (; t < nt; t += dt, hh += dh) {
    if (hh >= heads) {
      hh -= heads;
      if (++t >= nt) break;
    }
    const int side = hh >= a.heads[0], h = side ? hh - a.heads[0] : hh;
    rotate_unit<E>(a.x[side] + s_x[t][side] + h * a.xs[side][2],
                   a.y[side] + s_y[t][side] + h * a.ys[side][2], u, cs + t * slots, r2,
                   a.rot.interleaved != 0);
  }
}

}  // namespace fa
