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
__device__ __forceinline__ void unpack8(u32x4 raw, F *x) {
  const vec8<E> v = __builtin_bit_cast(vec8<E>, raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (F)(float)v[i];
}

__device__ __forceinline__ u32x4 load_raw8(const f16 *p) { return *reinterpret_cast<const u32x4 *>(p); }

// Place of pair j in a row's table of cosines and sines in LDS: lanes that own
// consecutive chunks of 8 columns read consecutive entries.
__device__ __forceinline__ int pair_slot(int j, int r2) { return (j & 7) * ((r2 + 7) >> 3) + (j >> 3); }
// Entries of a row's table.
__host__ __device__ __forceinline__ int pair_slots(int r2) { return 8 * ((r2 + 7) >> 3); }

// Offset of the chunk that holds the partners of columns 8c .. 8c+7, where they
// are one aligned chunk (half layout, R % 16 = 0, c in the rotated columns); 8c
// itself elsewhere.
__device__ __forceinline__ int partner_chunk(int c, int r2, bool interleaved) {
  const int d = 8 * c;
  if (interleaved || (r2 & 7) != 0 || d >= 2 * r2) return d;
  return d < r2 ? d + r2 : d - r2;
}

// Columns 8c .. 8c+7 of a row (`raw`), rotated by the row's table cs; `other` is
// partner_chunk's.  A lane then owns 8 consecutive columns whatever R is, and
// groups of 4 lanes the 32-column blocks that the 4-bit cache shares a scale
// over.  Partners that are no aligned chunk are loaded one by one; the branches
// but d < R are uniform.
template <typename E, typename F>
__device__ __forceinline__ void rotate8(u32x4 raw, u32x4 other, const f16 *row, int c,
                                        const CosSin<F> *cs, int r2, bool interleaved, F *y) {
  F x[8];
  unpack8<E, F>(raw, x);
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
      unpack8<E, F>(other, z);
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
__device__ __forceinline__ u32x4 pack8(const float *y) {
  vec8<E> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (E)y[i];
  return __builtin_bit_cast(u32x4, v);
}

__device__ __forceinline__ void store_raw8(f16 *p, u32x4 v) { *reinterpret_cast<u32x4 *>(p) = v; }

// Units of a row, one lane's work each: two chunks of 8 columns (one in rows of
// an odd number of chunks).  In the half layout with R % 16 = 0 the two are each
// other's partners, so that each is loaded, and its cosines read, once.
__host__ __device__ __forceinline__ int rotary_units(int D) { return D % 16 ? D / 8 : D / 16; }

struct RotaryUnit {
  int c0, c1;        // chunks; c1 = -1: none
  bool pair;
  __device__ __forceinline__ RotaryUnit(int u, int r2, bool interleaved, int D) {
    const int pairs = r2 >> 3;
    const bool half = !interleaved && (r2 & 7) == 0;
    pair = half && D % 16 == 0 && u < pairs;
    c0 = D % 16 ? u : (pair ? u : 2 * u);
    c1 = D % 16 ? -1 : (pair ? u + pairs : 2 * u + 1);
  }
};

// Rotates unit `u` of rows first, first + (dt, dh), .. of nt tokens x heads:
// in(t, h) and out(t, h) give a row's place, `ready` waits for the tables cs + t *
// slots.  2 rows' loads are in flight at a time, the first before the wait: a row
// is a few hundred bytes, and one at a time the sweep would wait for each.
template <typename E, typename In, typename Out, typename Ready>
__device__ __forceinline__ void rotate_rows(const RotaryUnit u, bool active, int t, int h, int dt,
                                            int dh, int nt, int heads, const CosSin<float> *cs,
                                            int slots, int r2, bool interleaved, In &&in,
                                            Out &&out, Ready &&ready) {
  constexpr int N = 2;
  bool waited = false;
  if (!active) t = nt;
  do {
    u32x4 x[N], z[N];
    int ts[N], hs[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (h >= heads) {
        h -= heads;
        ++t;
      }
      ts[j] = t;
      hs[j] = h;
      if (t < nt) {
        const f16 *row = in(t, h);
        x[j] = load_raw8(row + 8 * u.c0);
        if (u.c1 >= 0) z[j] = load_raw8(row + 8 * u.c1);
      }
      t += dt;
      h += dh;
    }
    if (!waited) ready();
    waited = true;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (ts[j] >= nt) break;
      const CosSin<float> *c = cs + ts[j] * slots;
      f16 *to = out(ts[j], hs[j]);
      if (u.pair) {
        float a[8], b[8], y[8];
        unpack8<E, float>(x[j], a);
        unpack8<E, float>(z[j], b);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const CosSin<float> v = c[u.c0 + i * (r2 >> 3)];
          y[i] = a[i] * v.c - b[i] * v.s;
          b[i] = b[i] * v.c + a[i] * v.s;
        }
        store_raw8(to + 8 * u.c0, pack8<E>(y));
        store_raw8(to + 8 * u.c1, pack8<E>(b));
      } else {
        // chunks behind R are copied as they are
        const f16 *row = in(ts[j], hs[j]);
#pragma unroll 1
        for (int k = 0; k < (u.c1 >= 0 ? 2 : 1); ++k) {
          const int chunk = k ? u.c1 : u.c0;
          u32x4 raw = k ? z[j] : x[j];
          if (8 * chunk < 2 * r2) {
            float y[8];
            rotate8<E, float>(raw, load_raw8(row + partner_chunk(chunk, r2, interleaved)), row,
                              chunk, c, r2, interleaved, y);
            raw = pack8<E>(y);
          }
          store_raw8(to + 8 * chunk, raw);
        }
      }
    }
  } while (t < nt);
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
  int S, D, unit_shift;   // log2 of the lanes for a row's units
  int64_t tokens;       // B * S
};

// One workgroup rotates every head of TOK tokens (or, split over gridDim.y,
// part of them).  Bound by HBM: each element is read and written once.  The
// cosines and sines of a token are shared by its heads: computed once per
// workgroup into LDS, then read by one lane per unit.  Lanes keep their unit and
// walk the (token, head) rows, so that the sweep has no division.
// 4096 tokens of 40 heads of 128, bf16: 17.3 us, 4.9 TB/s, the rate of a large
// copy (28 us with each column chunk loaded twice and an index divided a row);
// 32 tokens: 3.5 us, launch and two load latencies.
constexpr int kRotaryThreads = 256;

__device__ __forceinline__ int64_t rotary_position(const void *positions, int pos64, int64_t i) {
  return pos64 ? static_cast<const int64_t *>(positions)[i]
               : (int64_t) static_cast<const int32_t *>(positions)[i];
}

template <typename E, int TOK>
__global__ __launch_bounds__(kRotaryThreads) void fa_rotary_kernel(RotaryArgs a) {
  extern __shared__ char smem[];
  CosSin<float> *cs = reinterpret_cast<CosSin<float> *>(smem);   // [TOK][pair_slots]
  __shared__ int64_t s_x[TOK][2], s_y[TOK][2], s_p[TOK];         // a token's offsets
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
    s_p[tid] = b * a.pb + s * a.ps;
  }
  __syncthreads();
  const int u = tid & ((1 << a.unit_shift) - 1), lanes = kRotaryThreads >> a.unit_shift;
  const int heads = a.heads[0] + a.heads[1], step = lanes * gridDim.y;
  const int dt = step / heads, first = blockIdx.y * lanes + (tid >> a.unit_shift);
  const int t0 = first / heads;
  auto side = [&](int h) { return h >= a.heads[0] ? 1 : 0; };
  rotate_rows<E>(
      RotaryUnit(u, r2, a.rot.interleaved, a.D), u < rotary_units(a.D), t0, first - t0 * heads, dt,
      step - dt * heads, nt, heads, cs, slots, r2, a.rot.interleaved != 0,
      [&](int t, int h) {
        const int i = side(h);
        return a.x[i] + s_x[t][i] + (h - (i ? a.heads[0] : 0)) * a.xs[i][2];
      },
      [&](int t, int h) {
        const int i = side(h);
        return a.y[i] + s_y[t][i] + (h - (i ? a.heads[0] : 0)) * a.ys[i][2];
      },
      [&] {
        for (int i = tid; i < nt * r2; i += kRotaryThreads) {
          const int t = i / r2, j = i - t * r2;
          const int64_t p = rotary_position(a.positions, a.pos64, s_p[t]);
          CosSin<float> v = rotary_cos_sin<float>(p, a.rot.steps[j], (float)a.rot.factor);
          if (a.rot.inverse) v.s = -v.s;
          cs[t * slots + pair_slot(j, r2)] = v;
        }
        __syncthreads();
      });
}

}  // namespace fa
