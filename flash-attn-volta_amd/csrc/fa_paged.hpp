// fa_paged.hpp -- a paged key/value cache held in 4 bits: append, read back
// and the attention over it.
//
// Elements are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), 32 along D to a
// power of two: exponent floor(log2 max|x|) - 2, held + 127 in a byte.  Both
// conversions are one instruction a pair on this GPU (v_cvt_scalef32_pk_*_fp4,
// v_cvt_scalef32_pk_fp4_f32) and every value is exact in bf16, and in fp16
// from 2^-24 up, so the attention's products see what the cache holds.
//
// Page layout (N pages, Hk heads, P tokens, P a power of two >= 16):
//   k_codes  [N][Hk][P][D/2]           a token's row, even d in the low half
//   k_scales [N][Hk][P][D/32]
//   v_codes  [N][Hk][P/4][16][4][D/32] token 4a + r, d = (D/16) m + j
//   v_scales [N][Hk][P/4][D/32][4]
// K rows are the A operand's rows of S^T = K Q^T: a lane's 8 columns of one
// key.  V is the A operand of O^T = V^T P^T, where a lane needs several keys
// of one column: with 4 tokens interleaved the 4 keys that a lane's result
// registers of S^T hold are the 4 keys of its next 16-byte V load, so
// probabilities go from one product to the next in registers and nothing
// passes through LDS; a token's codes stay whole bytes of its own, so appending
// one touches no other.
//
// The cache holds finite values only: infinities are stored as the largest
// that fits, NaN as 0.  What unseen slots hold can then meet a probability of
// 0 without making it a NaN, and stale pages need no clearing.
#pragma once

#include "fa_common.hpp"
#include "fa_rotary.hpp"

namespace fa {

struct PagedCache {
  uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const int32_t *table;   // (B, width), row stride width_stride
  int64_t table_stride;
  int n_pages, width;
  int page_shift;         // log2 P
  int Hk;
};

// Page of position `pos` of sequence b, or -1 (outside the table, or an id
// that is no page: such slots hold nothing and take nothing).
__device__ __forceinline__ int page_of(const PagedCache &c, int b, int64_t pos) {
  if (pos < 0 || (pos >> c.page_shift) >= c.width) return -1;
  const int id = c.table[b * c.table_stride + (pos >> c.page_shift)];
  return (unsigned)id < (unsigned)c.n_pages ? id : -1;
}

// Row (page, h, slot) of k_codes in rows of D/2 bytes; the same index times
// D/32 is its first scale.
__device__ __forceinline__ int64_t paged_row(const PagedCache &c, int page, int h, int slot) {
  return ((((int64_t)page * c.Hk + h) << c.page_shift) + slot);
}

__device__ __forceinline__ float fp4_scale(unsigned byte) { return __uint_as_float(byte << 23); }

// -- append --------------------------------------------------------------------

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 8;   // positions 8a .. 8a + 7 to a workgroup

struct AppendArgs {
  PagedCache cache;
  const f16 *k, *v, *q;
  f16 *q_out;
  int64_t ks[3], vs[3], qs[3], qos[3];   // {b, s, h}
  const int32_t *start, *counts;         // counts: NULL = S everywhere
  RotaryTable rot;                       // steps NULL: no rotation
  int S, H;
  int parts;                             // of gridDim.y, those that store keys and values
  int unit_shift;                        // log2 of the lanes for a row of q
  float top;                             // largest finite value that is kept
  int max_byte;                          // largest scale byte
};

// fp32 of x for a later rounding to few bits: inexact results get an odd last
// bit (rounding to odd), so that the two roundings are as one.
__device__ __forceinline__ float odd_float(double x) {
  float f = (float)x;
  const double d = (double)f;
  if (d != x && __builtin_isfinite(f)) {
    uint32_t u = __float_as_uint(f);
    if (!(u & 1)) u += (fabs(d) < fabs(x)) ? 1u : ~0u;
    f = __uint_as_float(u);
  }
  return f;
}

// Codes and scale byte of 8 of a block's 32 columns; the block's other 24 are
// in the three adjacent lanes.
__device__ __forceinline__ uint32_t quantise8(float *y, float top, int max_byte, unsigned &byte) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = y[i] != y[i] ? 0.0f : fminf(fmaxf(y[i], -top), top);
    m = fmaxf(m, fabsf(y[i]));
  }
  // (quad_perm [1, 0, 3, 2], then [2, 3, 0, 1]; m >= 0 orders as its bits)
  m = __uint_as_float(dpp_umax<0x4E, 0xF>(dpp_umax<0xB1, 0xF>(__float_as_uint(m))));
  byte = (unsigned)min(max((int)(__float_as_uint(m) >> 23) - 2, 1), max_byte);
  const float s = fp4_scale(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], s, 3);
  return w;
}

// Workgroup (tile, part, b): the new tokens at positions 8a .. 8a + 7 of
// sequence b; the first parts of a tile store keys and values, the rest rotate q.
// Keys are rotated in fp64, from cosines and sines computed once a token in LDS: a
// code is the nearest to the rotated value itself, so the same key at the same
// position gets the same code whichever path computed it.  q is rotated in
// fp32, as fa_rotary does.  Consecutive lanes are the D/8 chunks of a key's
// row, then the tokens, whose 4-byte pieces of an interleaved V group then fill
// whole lines.  Bound by HBM on prompts and by launch and load latency on single
// tokens: 6001 tokens of 32 / 8 heads of 128 with q, 32.4 us, 4.0 TB/s (80 % of a
// large copy's rate); one token 3.5 us.
template <typename E, int D>
__global__ __launch_bounds__(kAppendThreads) void fa_paged_append_kernel(AppendArgs a) {
  extern __shared__ char smem[];
  constexpr int NCH = D / 8;
  const int r2 = a.rot.steps ? a.rot.r2 : 0, slots = pair_slots(r2);
  const int b = blockIdx.z, tid = threadIdx.x;
  const int64_t start = a.start[b];
  // tokens i0 .. i0 + nt - 1 of this tile
  const int64_t base = (start & ~(int64_t)(kAppendTokens - 1)) + (int64_t)blockIdx.x * kAppendTokens;
  const int i0 = (int)max((int64_t)0, base - start);
  int nt = (int)(min((int64_t)a.S, base + kAppendTokens - start) - i0);
  if ((int)blockIdx.y >= a.parts) {
    // queries (rows behind the count too: they are results, not cache)
    if (nt <= 0) return;
    CosSin<float> *cs = reinterpret_cast<CosSin<float> *>(smem);
    const int u = tid & ((1 << a.unit_shift) - 1), lanes = kAppendThreads >> a.unit_shift;
    const int step = lanes * (gridDim.y - a.parts), dt = step / a.H;
    const int first = (blockIdx.y - a.parts) * lanes + (tid >> a.unit_shift), t0 = first / a.H;
    const f16 *q = a.q + b * a.qs[0] + (int64_t)i0 * a.qs[1];
    f16 *out = a.q_out + b * a.qos[0] + (int64_t)i0 * a.qos[1];
    rotate_rows<E>(
        RotaryUnit(u, r2, a.rot.interleaved, D), u < rotary_units(D), t0, first - t0 * a.H, dt,
        step - dt * a.H, nt, a.H, cs, slots, r2, a.rot.interleaved != 0,
        [&](int t, int h) { return q + t * a.qs[1] + h * a.qs[2]; },
        [&](int t, int h) { return out + t * a.qos[1] + h * a.qos[2]; },
        [&] {
          for (int i = tid; i < nt * r2; i += kAppendThreads) {
            const int t = i / r2, j = i - t * r2;
            cs[t * slots + pair_slot(j, r2)] =
                rotary_cos_sin<float>(start + i0 + t, a.rot.steps[j], (float)a.rot.factor);
          }
          if (r2) __syncthreads();
        });
    return;
  }
  if (a.counts) nt = min(nt, max(a.counts[b], 0) - i0);
  if (nt <= 0) return;
  CosSin<double> *cs = reinterpret_cast<CosSin<double> *>(smem);
  // 8 aligned positions are slots of one page
  const int64_t pos0 = start + i0;
  const int page = page_of(a.cache, b, pos0);
  const int slot0 = (int)(pos0 & ((1 << a.cache.page_shift) - 1));
  // Lane: chunk c of rows first, first + (dt, dh), ..: token t of head h.
  // Whole blocks of 32 columns stay together, in groups of 4 lanes.
  constexpr int kRows = kAppendThreads / NCH;
  const int Hk = a.cache.Hk, c = tid % NCH, step = kRows * a.parts;
  const int dh = step / nt, dt = step - dh * nt;
  const int first = blockIdx.y * kRows + tid / NCH;
  int h = first / nt, t = first - h * nt;
  const f16 *k = a.k + b * a.ks[0] + (int64_t)i0 * a.ks[1], *v = a.v + b * a.vs[0] + (int64_t)i0 * a.vs[1];
  const int other = partner_chunk(c, r2, a.rot.interleaved != 0);
  u32x4 kx, kz, vx;                      // the next row's
  auto fetch = [&] {
    if (h < Hk) {
      const f16 *kr = k + t * a.ks[1] + h * a.ks[2];
      kx = load_raw8(kr + 8 * c);
      kz = load_raw8(kr + other);
      vx = load_raw8(v + t * a.vs[1] + h * a.vs[2] + 8 * c);
    }
  };
  fetch();
  for (int i = tid; i < nt * r2; i += kAppendThreads) {
    const int j = i / r2, p = i - j * r2;
    cs[j * slots + pair_slot(p, r2)] =
        rotary_cos_sin<double>(pos0 + j, a.rot.steps[p], a.rot.factor);
  }
  if (r2) __syncthreads();
  while (h < Hk) {
    const int ht = h, tt = t;
    float vy[8], ky[8];
    unpack8<E, float>(vx, vy);
    const u32x4 x = kx, z = kz;
    h += dh;
    t += dt;
    if (t >= nt) {
      t -= nt;
      ++h;
    }
    fetch();
    if (r2) {
      double y[8];
      rotate8<E, double>(x, z, k + tt * a.ks[1] + ht * a.ks[2], c, cs + tt * slots, r2,
                         a.rot.interleaved != 0, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) ky[j] = odd_float(y[j]);
    } else {
      unpack8<E, float>(x, ky);
    }
    unsigned kb, vb;
    const uint32_t kw = quantise8(ky, a.top, a.max_byte, kb);
    const uint32_t vw = quantise8(vy, a.top, a.max_byte, vb);
    if (page < 0) continue;
    const int64_t row = paged_row(a.cache, page, ht, slot0 + tt);
    *reinterpret_cast<uint32_t *>(a.cache.k_codes + row * (D / 2) + 4 * c) = kw;
    // group row / 4, token r = row % 4: unit m of a group is 4 tokens x D/32 bytes
    const int64_t group = row >> 2;
    const int r = (int)(row & 3);
    uint8_t *vp = a.cache.v_codes + group * (2 * D);
    if constexpr (D == 128) {
      *reinterpret_cast<uint32_t *>(vp + (c * 4 + r) * 4) = vw;
    } else if constexpr (D == 64) {
      *reinterpret_cast<uint16_t *>(vp + ((2 * c) * 4 + r) * 2) = (uint16_t)vw;
      *reinterpret_cast<uint16_t *>(vp + ((2 * c + 1) * 4 + r) * 2) = (uint16_t)(vw >> 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) vp[(4 * c + j) * 4 + r] = (uint8_t)(vw >> (8 * j));
    }
    if ((c & 3) == 0) {
      a.cache.k_scales[row * (D / 32) + c / 4] = (uint8_t)kb;
      a.cache.v_scales[(group * (D / 32) + c / 4) * 4 + r] = (uint8_t)vb;
    }
  }
}

// -- the values that codes stand for ------------------------------------------------

template <typename E> struct Fp4;

template <> struct Fp4<f16> {
  template <int BYTE> static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, BYTE));
  }
};

template <> struct Fp4<bf16> {
  template <int BYTE> static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, BYTE));
  }
};

// 8 values of a dword of codes.
template <typename E>
__device__ __forceinline__ u32x4 fp4_row8(uint32_t w, float s) {
  return u32x4{Fp4<E>::template pair<0>(w, s), Fp4<E>::template pair<1>(w, s),
               Fp4<E>::template pair<2>(w, s), Fp4<E>::template pair<3>(w, s)};
}

struct ReadArgs {
  PagedCache cache;
  f16 *k, *v;              // (B, n, Hk, D) contiguous
  const int32_t *start, *counts;
  int n;
  int64_t work;            // B * n * Hk * D / 8
};

// Tokens start[b] .. start[b] + n - 1 as 16-bit rows; 0 where nothing is held
// (behind counts[b], outside the table, on a page that is none).  Bound by HBM, by
// what it writes: 6001 tokens of 8 heads of 128 8.2 us (3.8 TB/s).
template <typename E, int D>
__global__ __launch_bounds__(256) void fa_paged_read_kernel(ReadArgs a) {
  constexpr int NCH = D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.work) return;
  const int Hk = a.cache.Hk;
  // chunk, then token, then head: 4 tokens of a V group in adjacent lanes
  const int c = (int)(i % NCH);
  int64_t rest = i / NCH;
  const int t = (int)(rest % a.n);
  rest /= a.n;
  const int h = (int)(rest % Hk), b = (int)(rest / Hk);
  u32x4 ko = {0, 0, 0, 0}, vo = {0, 0, 0, 0};
  const int64_t pos = (int64_t)a.start[b] + t;
  const int page = a.counts && t >= a.counts[b] ? -1 : page_of(a.cache, b, pos);
  if (page >= 0) {
    const int64_t row =
        paged_row(a.cache, page, h, (int)(pos & ((1 << a.cache.page_shift) - 1)));
    const int64_t group = row >> 2;
    const int r = (int)(row & 3);
    const uint32_t kw = *reinterpret_cast<const uint32_t *>(a.cache.k_codes + row * (D / 2) + 4 * c);
    const uint8_t *vp = a.cache.v_codes + group * (2 * D);
    uint32_t vw;
    if constexpr (D == 128) {
      vw = *reinterpret_cast<const uint32_t *>(vp + (c * 4 + r) * 4);
    } else if constexpr (D == 64) {
      vw = *reinterpret_cast<const uint16_t *>(vp + ((2 * c) * 4 + r) * 2) |
           (uint32_t) * reinterpret_cast<const uint16_t *>(vp + ((2 * c + 1) * 4 + r) * 2) << 16;
    } else {
      vw = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) vw |= (uint32_t)vp[(4 * c + j) * 4 + r] << (8 * j);
    }
    ko = fp4_row8<E>(kw, fp4_scale(a.cache.k_scales[row * (D / 32) + c / 4]));
    vo = fp4_row8<E>(vw, fp4_scale(a.cache.v_scales[(group * (D / 32) + c / 4) * 4 + r]));
  }
  const int64_t o = (((int64_t)b * a.n + t) * Hk + h) * D + 8 * c;
  *reinterpret_cast<u32x4 *>(a.k + o) = ko;
  *reinterpret_cast<u32x4 *>(a.v + o) = vo;
}

// -- attention ---------------------------------------------------------------------

__device__ __forceinline__ floatx4 mfma16(vec8<f16> a, vec8<f16> b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ floatx4 mfma16(vec8<bf16> a, vec8<bf16> b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

struct PagedAttnArgs {
  PagedCache cache;
  const f16 *q;
  int64_t qs[3];                        // {b, s, h}
  f16 *o;                               // (B, Sq, H, D) contiguous
  float *lse;                           // (B, H, Sq) or NULL
  const int32_t *lengths, *counts;      // counts: NULL = Sq everywhere
  float *part_o;                        // (target + 1, Hk, rows, D) unnormalised
  float *part_ml;                       // (target + 1, Hk, rows, 2): maximum (log2), sum
                                        // then, with B > 1, (B, 2) int: Chunk::count, part
  int B, Sq, H, G;
  int target;                           // chunks aimed at
  float c;                              // |sm_scale| log2 e
  uint32_t flip;                        // sign bits xor-ed into q (negative scale)
};

// A value that the kernel does not write, at an address that is the same in every lane.
__device__ __forceinline__ int scalar_load(const int32_t *p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(
      reinterpret_cast<uintptr_t>(p));
}

// Has these kernel arguments in registers at this point: they are loaded together,
// where the compiler would load each before its first use and wait for it there (one
// query on 4096 tokens, two kernels: 8.45 / 8.25 us).
template <typename T> __device__ __forceinline__ void have_one(T x) { asm volatile("" : : "s"(x)); }
template <typename... T> __device__ __forceinline__ void have(T... x) { (have_one(x), ...); }

// Queries of a packed tile: row n of (b, hk) is query n / G of head hk G + n % G.
// Keys a row sees: positions <= lengths - counts + query.
constexpr int kUnit = 128;              // keys: one step of the 4 waves
constexpr float kLowest = -3.4028234663852886e38f;

struct Chunk {
  int b, index, count, keys;            // `count` chunks of `keys` keys in sequence b
  int part;                             // partial result of its chunk 0, where count > 1
  int length, held;                     // lengths[b], and what of it the table holds
};

__device__ __forceinline__ int held_keys(const PagedAttnArgs &a, int length) {
  const int64_t cap = (int64_t)a.cache.width << a.cache.page_shift;
  return (int)max((int64_t)0, min((int64_t)length, cap));
}

// Inclusive prefix sum over the wave: within rows of 16 lanes (row_shr 1, 2, 4,
// 8; lanes without a source add 0), then each row's last into the rows behind
// (row_bcast 15, 31).
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}

__device__ __forceinline__ int wave_prefix(int x) {
  x = dpp_add<0x111, 0xF>(x);
  x = dpp_add<0x112, 0xF>(x);
  x = dpp_add<0x114, 0xF>(x);
  x = dpp_add<0x118, 0xF>(x);
  x = dpp_add<0x142, 0xA>(x);
  return dpp_add<0x143, 0xC>(x);
}

__device__ __forceinline__ int units_of(int held) { return (held + kUnit - 1) / kUnit; }

// ceil(u / units), 1 at least, u and units up to 2^23: an fp32 quotient, off by
// one at most.
__device__ __forceinline__ int parts(int u, int units) {
  const int x = u + units - 1;
  int q = (int)((float)x * __builtin_amdgcn_rcpf((float)units));
  q -= q * units > x ? 1 : 0;
  q += (q + 1) * units <= x ? 1 : 0;
  return max(1, q);
}

// The chunks of a batch of one sequence (one user's tokens: scalar work alone).
__device__ __forceinline__ void one_sequence(const PagedAttnArgs &a, Chunk &out) {
  out.b = out.part = 0;
  out.length = scalar_load(a.lengths);
  out.held = held_keys(a, out.length);
  const int u = units_of(out.held), units = parts(u, a.target);
  out.count = parts(u, units);
  out.keys = units * kUnit;
}

// Splits all sequences' keys evenly: chunks of the same whole number of units
// (the last of a sequence shorter), `target` of them at most where that can be,
// whatever the lengths.  The host knows no lengths; every wave counts them for
// itself (B loads) and finds the sequence of its slot; one that holds nothing is
// a chunk too, which writes its zeros.  max(target, (target + 1) / 2 + B) slots
// cover every chunk, B with a target of 1 (then no sequence is split); those of
// sequences that are split are target + 1 at most (n > 1 chunks are under twice
// their units' share).  The first chunk of each of several sequences leaves its count for
// the join, which would be longer over finding it than over joining (us with a join that
// counts: 32 sequences on up to 3001 tokens 19.8, now 19.3, 128 on 4000 109, now 105;
// a single sequence, which needs no counting, would lose 0.3).
__device__ __forceinline__ bool find_chunk(const PagedAttnArgs &a, int want, Chunk &out) {
  const int lane = threadIdx.x & 63;
  if (a.target == 1) {                  // nothing is split: a slot is a sequence
    out.b = want;
    out.index = out.part = 0;
    out.count = 1;
    out.length = scalar_load(a.lengths + want);
    out.held = held_keys(a, out.length);
    out.keys = 1 << 30;
    return true;
  }
  if (a.B == 1) {
    one_sequence(a, out);
    out.index = want;
    return want < out.count;
  }
  // Units of a chunk.  (2^23 are a whole sequence of any length; more of them, in a
  // batch of over 2^31 keys, would leave the range of positions.)
  auto share = [&](int total, int chunks) {
    return min(max(1, (total - 1) / chunks + 1), 1 << 23);
  };
  // Short last chunks can go over the target: then as many fewer whole ones as there
  // are sequences, half the target at least.
  auto fewer = [&](int total) { return share(total, max(a.target - a.B, (a.target + 1) / 2)); };
  int length = 0, held = 0;
  auto load = [&](int b) {              // units of sequence b, this lane's
    length = b < a.B ? a.lengths[b] : 0;
    held = held_keys(a, length);
    return units_of(held);
  };
  // Prefix sums of the chunks and of those of split sequences: two 16-bit halves,
  // under 2^15 both (targets are workgroups of one round, 64 sequences a time).
  auto prefix = [&](int n) { return wave_prefix(n | (n > 1 ? n << 16 : 0)); };
  auto find = [&](int upto, int n, int b0, int before, int before_split, int units) {
    const int first = before + (upto & 0xFFFF) - n;
    const bool mine = want >= first && want < first + n;
    const uint64_t hit = __ballot(mine);
    if (!hit) return false;
    const int src = __builtin_ctzll(hit);
    out.b = b0 + src;
    out.count = __builtin_amdgcn_readlane(n, src);
    out.part = before_split + __builtin_amdgcn_readlane((upto >> 16) - n, src);
    out.length = __builtin_amdgcn_readlane(length, src);
    out.held = __builtin_amdgcn_readlane(held, src);
    out.index = want - __builtin_amdgcn_readlane(first, src);
    out.keys = units * kUnit;
    return true;
  };
  auto last = [](int x) { return __builtin_amdgcn_readlane(x, 63); };
  if (a.B <= 64) {
    const int u = load(lane), total = last(wave_prefix(u));
    int units = share(total, a.target);
    int n = lane < a.B ? parts(u, units) : 0, upto = prefix(n);
    if ((last(upto) & 0xFFFF) > a.target) {
      units = fewer(total);
      n = lane < a.B ? parts(u, units) : 0;
      upto = prefix(n);
    }
    return find(upto, n, 0, 0, 0, units);
  }
  // 4 groups of 64 sequences at a time, their loads in flight together
  constexpr int kGroups = 4;
  int group[kGroups];
  auto load_groups = [&](int b0) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int b = b0 + 64 * j + lane;
      group[j] = b < a.B ? a.lengths[b] : 0;
    }
  };
  auto sum = [&](auto &&f) {            // over all sequences
    int x = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64 * kGroups) {
      load_groups(b0);
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
        x += b0 + 64 * j + lane < a.B ? f(units_of(held_keys(a, group[j]))) : 0;
    }
    return last(wave_prefix(x));
  };
  const int total = sum([](int u) { return u; });
  int units = share(total, a.target);
  if (sum([&](int u) { return parts(u, units); }) > a.target) units = fewer(total);
  int before = 0, before_split = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64 * kGroups) {
    load_groups(b0);
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int at = b0 + 64 * j;
      length = group[j];
      held = held_keys(a, length);
      const int n = at + lane < a.B ? parts(units_of(held), units) : 0, upto = prefix(n);
      if (find(upto, n, at, before, before_split, units)) return true;
      before += last(upto) & 0xFFFF;
      before_split += last(upto) >> 16;
    }
  }
  return false;
}

__device__ __forceinline__ int *chunk_counts(const PagedAttnArgs &a) {
  return reinterpret_cast<int *>(a.part_ml + (int64_t)(a.target + 1) * a.cache.Hk * (a.Sq * a.G) * 2);
}

// (by the first workgroup of a sequence, where any may be split)
__device__ __forceinline__ void leave_count(const PagedAttnArgs &a, const Chunk &ch, int hk) {
  if (a.B > 1 && a.target > 1 && ch.index == 0 && (hk | blockIdx.y | threadIdx.x) == 0) {
    int *to = chunk_counts(a) + 2 * ch.b;
    to[0] = ch.count;
    to[1] = ch.part;
  }
}

template <int D> struct KRaw { u32x4 w; };
template <> struct KRaw<64> { u32x2 w; };
template <> struct KRaw<32> { uint32_t w; };

template <int D> __device__ __forceinline__ uint32_t raw_word(const KRaw<D> &r, int i) { return r.w[i]; }
template <> __device__ __forceinline__ uint32_t raw_word<32>(const KRaw<32> &r, int) { return r.w; }

// One wave's share of a 16-key tile: codes of key m's quarter g of the columns
// and of V group g's unit m, each with its scales.
template <int D> struct Tile16 {
  KRaw<D> k, v;
  uint32_t ks, vs;
  bool hole;
};

// Row of 16-key tile `key` in its page, and whether it is a hole: no key, or a page
// that is none (page 0 is read instead, its keys masked).
__device__ __forceinline__ int64_t tile_row(const PagedCache &c, int b, int hk, int key, int end,
                                            bool &hole) {
  // (the id is loaded whether it is needed or not: no branch in the sweeps)
  const int page = scalar_load(c.table + b * c.table_stride + min(key >> c.page_shift, c.width - 1));
  hole = key >= end || (unsigned)page >= (unsigned)c.n_pages;
  return paged_row(c, hole ? 0 : page, hk, key & ((1 << c.page_shift) - 1));
}

template <int D>
__device__ __forceinline__ void load_k(const PagedCache &c, int64_t row, int m, int g, Tile16<D> &t) {
  t.k = *reinterpret_cast<const KRaw<D> *>(c.k_codes + row * (D / 2) + m * (D / 2) + g * (D / 8));
  t.ks = (c.k_scales + row * (D / 32))[m * (D / 32) + g * D / 128];
}

template <int D>
__device__ __forceinline__ void load_v(const PagedCache &c, int64_t row, int m, int g, Tile16<D> &t) {
  t.v = *reinterpret_cast<const KRaw<D> *>(c.v_codes + row * (D / 2) + (g * 16 + m) * (D / 8));
  t.vs = *reinterpret_cast<const uint32_t *>(c.v_scales + row * (D / 32) +
                                             (g * (D / 32) + m * D / 512) * 4);
}

template <int D>
__device__ __forceinline__ void load_tile(const PagedCache &c, int b, int hk, int key, int end,
                                          int m, int g, Tile16<D> &t) {
  const int64_t row = tile_row(c, b, hk, key, end, t.hole);
  load_k<D>(c, row, m, g, t);
  load_v<D>(c, row, m, g, t);
}

// Byte pair s of key r in a V unit: the codes of d = 2s, 2s + 1 of the unit.
template <typename E, int D, int S>
__device__ __forceinline__ uint32_t v_pair(const KRaw<D> &v, int r, float scale) {
  // (r is a constant after unrolling)
  if constexpr (D == 128) {
    return Fp4<E>::template pair<S>(v.w[r], scale);
  } else if constexpr (D == 64) {
    return (r & 1) ? Fp4<E>::template pair<S + 2>(v.w[r >> 1], scale)
                   : Fp4<E>::template pair<S>(v.w[r >> 1], scale);
  } else {
    return r == 0   ? Fp4<E>::template pair<0>(v.w, scale)
           : r == 1 ? Fp4<E>::template pair<1>(v.w, scale)
           : r == 2 ? Fp4<E>::template pair<2>(v.w, scale)
                    : Fp4<E>::template pair<3>(v.w, scale);
  }
}

// O^T tiles 2S and 2S + 1 += V^T P^T over 32 keys.
template <typename E, int D, int NT, int PARTS, int S>
__device__ __forceinline__ void pv_step(const Tile16<D> (&t)[2], const float (&vsc)[2][4],
                                        const vec8<E> (&p)[PARTS][NT], floatx4 (&o)[NT][D / 16]) {
  u32x4 lo, hi;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      const uint32_t x = v_pair<E, D, S>(t[u].v, r, vsc[u][r]);
      const uint32_t y = v_pair<E, D, S>(t[u].v, r + 1, vsc[u][r + 1]);
      lo[2 * u + r / 2] = __builtin_amdgcn_perm(y, x, 0x05040100u);
      hi[2 * u + r / 2] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    }
  const vec8<E> a0 = __builtin_bit_cast(vec8<E>, lo), a1 = __builtin_bit_cast(vec8<E>, hi);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      o[nt][2 * S] = mfma16(a0, p[q][nt], o[nt][2 * S]);
      o[nt][2 * S + 1] = mfma16(a1, p[q][nt], o[nt][2 * S + 1]);
    }
  if constexpr (S + 1 < D / 32) pv_step<E, D, NT, PARTS, S + 1>(t, vsc, p, o);
}

// Few query rows (decode): workgroup (slot x head, row tile of 16 NT rows), 4
// waves, each sweeping every fourth 32-key step of the chunk on its own with
// its own running maximum; joined through LDS at the end.  Bound by reading the
// cache: no LDS, barrier or shuffle in the sweep, the next step's codes in
// flight while one is computed.  Lane (m, g) = (lane % 16, lane / 16).
// bf16 probabilities go into the product as two bf16 numbers whose sum has 16
// bits: the extra MFMAs hide behind the loads, and a single one would add a
// rounding as large as the output's own.
// 2 users' tokens on 131072 of 32 / 8 heads of 128: 51.6 us, 5.5 TB/s (a large copy
// runs at 4.9); 32 on up to 3001: 15.7 us, 4.2 TB/s; one on 4096: 4.8 us, a launch
// and three dependent loads (length, page, codes).  Vector instructions take 60 %
// of the cycles, half of them conversions, matrix ones 12 %.
template <typename E, int D, int NT>
__global__ __launch_bounds__(256) void fa_paged_few_kernel(PagedAttnArgs a) {
  constexpr int KS = D / 32, ND = D / 16, NW = 4;
  constexpr int PARTS = std::is_same<E, bf16>::value ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = a.cache.Hk, hk = blockIdx.x % Hk, slot = blockIdx.x / Hk;
  have(a.cache.k_codes, a.cache.k_scales, a.cache.v_codes, a.cache.v_scales, a.cache.table,
       a.cache.table_stride, a.cache.n_pages, a.cache.width);
  Chunk ch;
  if (!find_chunk(a, slot, ch)) return;
  const int b = ch.b, rows = a.Sq * a.G, row0 = blockIdx.y * (16 * NT);
  const int held = ch.held;
  const int count = a.counts ? min(max(scalar_load(a.counts + b), 0), a.Sq) : a.Sq;
  const int base = ch.length - count;             // position of query 0

  // Q as B operands: column n = row0 + 16 nt + m, d = (D/4) g + 8 t + 0..7
  vec8<E> qf[NT][KS];
  int last[NT];                                   // last position that the row sees
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = row0 + 16 * nt + m, i = n / a.G;
    const bool real = n < rows && i < count;
    last[nt] = real ? base + i : -1;
    const f16 *qp = a.q + b * a.qs[0] + (int64_t)(real ? i : 0) * a.qs[1] +
                    (hk * a.G + (real ? n - i * a.G : 0)) * a.qs[2] + (D / 4) * g;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      u32x4 raw = *reinterpret_cast<const u32x4 *>(qp + 8 * t);
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j] = real ? raw[j] ^ a.flip : 0u;
      qf[nt][t] = __builtin_bit_cast(vec8<E>, raw);
    }
  }
  // the tile's rows see every key below `all`, none from `end` on
  const int i_first = row0 / a.G, i_last = min((row0 + 16 * NT - 1) / a.G, count - 1);
  const int all = base + i_first + 1;
  const int key0 = ch.index * ch.keys;
  const int end = i_first < count ? min(min(held, key0 + ch.keys), base + i_last + 1) : 0;

  float mx[NT], l[NT];
  floatx4 o[NT][ND];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    mx[nt] = kLowest;
    l[nt] = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t) o[nt][t] = floatx4{0, 0, 0, 0};
  }

  Tile16<D> cur[2], nxt[2];
  int key = key0 + 32 * w;
  if (key < end) {
#pragma unroll
    for (int u = 0; u < 2; ++u) load_tile<D>(a.cache, b, hk, key + 16 * u, end, m, g, nxt[u]);
  }
  for (; key < end; key += 32 * NW) {
#pragma unroll
    for (int u = 0; u < 2; ++u) cur[u] = nxt[u];
    const int ahead = key + 32 * NW;
    if (ahead < end) {
#pragma unroll
      for (int u = 0; u < 2; ++u) load_tile<D>(a.cache, b, hk, ahead + 16 * u, end, m, g, nxt[u]);
    }
    // S^T: rows (keys) 4g + i of each 16-key tile, column (query) m
    floatx4 s[2][NT];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float sc = fp4_scale(cur[u].ks);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[u][nt] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const vec8<E> kf = __builtin_bit_cast(vec8<E>, fp4_row8<E>(raw_word<D>(cur[u].k, t), sc));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[u][nt] = mfma16(kf, qf[nt][t], s[u][nt]);
      }
    }
    if (key + 32 > all || key + 32 > end || cur[0].hole || cur[1].hole) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = key + 16 * u + 4 * g + i;
            if (cur[u].hole || kk >= end || kk > last[nt]) s[u][nt][i] = kNegInf;
          }
    }
    vec8<E> p[PARTS][NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = s[0][nt][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i >> 2][nt][i & 3]);
      top *= a.c;
      // a new maximum only for rows whose old one is left behind by 2^8: no row's
      // rounding depends on the other rows of its tile
      if (__any(top > mx[nt] + 8.0f)) {
        float t = fmaxf(top, __shfl_xor(top, 16, 64));
        t = fmaxf(t, xor32(t));
        t = t > mx[nt] + 8.0f ? t : mx[nt];
        const float f = fast_exp2(mx[nt] - t);
        mx[nt] = t;
        l[nt] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[nt][d] *= f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = fast_exp2(s[i >> 2][nt][i & 3] * a.c - mx[nt]);
        l[nt] += e;
        p[0][nt][i] = (E)e;
        if constexpr (PARTS == 2) p[1][nt][i] = (E)(e - (float)p[0][nt][i]);
      }
    }
    float vsc[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) vsc[u][r] = fp4_scale((cur[u].vs >> (8 * r)) & 0xFFu);
    pv_step<E, D, NT, PARTS, 0>(cur, vsc, p, o);
  }

  // Join the waves.  O^T tile t, register i: column (query) m, d = (D/16)(4g + i) + t.
  __shared__ float s_o[NW][NT][D][17];            // 17: columns of a row in different banks
  __shared__ float s_m[NW][16 * NT], s_l[NW][16 * NT];
  const int here = min(rows - row0, 16 * NT);     // rows of this tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float ls = l[nt] + __shfl_xor(l[nt], 16, 64);
    ls += xor32(ls);
    if (16 * nt + m < here) {
      if (g == 0) {
        s_m[w][16 * nt + m] = mx[nt];
        s_l[w][16 * nt + m] = ls;
      }
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_o[w][nt][ND * (4 * g + i) + t][m] = o[nt][t][i];
    }
  }
  __syncthreads();
  // a row to every 256 / 2^k threads, 2^k >= rows: its factors once a thread
  const int lanes = 256 >> (here > 1 ? 32 - __builtin_clz(here - 1) : 0);
  const int n = tid / lanes, row = row0 + n;
  if (n >= here) return;
  const int i = row / a.G, h = hk * a.G + (row - i * a.G);
  float top = s_m[0][n], sum = 0.0f, f[NW];
#pragma unroll
  for (int k = 1; k < NW; ++k) top = fmaxf(top, s_m[k][n]);
#pragma unroll
  for (int k = 0; k < NW; ++k) {
    f[k] = fast_exp2(s_m[k][n] - top);
    sum += s_l[k][n] * f[k];
  }
  const bool real = i < count, whole = ch.count == 1;
  const float inv = !real || sum == 0.0f ? 0.0f : (whole ? 1.0f / sum : 1.0f);   // (NaN: kept)
  const int64_t part = ((int64_t)(ch.part + ch.index) * Hk + hk) * rows + row;
  const int64_t out = (((int64_t)b * a.Sq + i) * a.H + h) * D;
  // columns in groups of 4 where each thread has as many, else one by one (us: 16 x 4
  // queries of 14 / 2 heads of 64 on up to 5000 tokens 12.3 / 12.7, 100 x 4 of 32 / 8 of
  // 128 on up to 500 13.6 / 14.2; 64 x 1 of 16 / 16 of 64 on up to 1500 17.8 / 17.4)
  auto leave = [&](auto W) {
    constexpr int kw = decltype(W)::value;
    typedef float F __attribute__((ext_vector_type(kw)));
    typedef E X __attribute__((ext_vector_type(kw)));
    for (int d = kw * (tid % lanes); d < D; d += kw * lanes) {
      F acc = 0.0f;
#pragma unroll
      for (int k = 0; k < NW; ++k)
#pragma unroll
        for (int j = 0; j < kw; ++j) acc[j] += s_o[k][n >> 4][d + j][n & 15] * f[k];
      X x;
#pragma unroll
      for (int j = 0; j < kw; ++j) {
        acc[j] = inv == 0.0f ? 0.0f : acc[j] * inv;
        x[j] = (E)acc[j];
      }
      if (whole)
        *reinterpret_cast<X *>(reinterpret_cast<E *>(a.o) + out + d) = x;
      else
        *reinterpret_cast<F *>(a.part_o + part * D + d) = acc;
    }
  };
  if (4 * lanes <= D)
    leave(std::integral_constant<int, 4>{});
  else
    leave(std::integral_constant<int, 1>{});
  if (tid % lanes != 0) return;
  leave_count(a, ch, hk);
  if (!whole) {
    a.part_ml[part * 2] = top;
    a.part_ml[part * 2 + 1] = real ? sum : 0.0f;
  } else if (a.lse) {
    a.lse[((int64_t)b * a.H + h) * a.Sq + i] =
        !real || sum == 0.0f ? kPosInf : (top + fast_log2(sum)) * kLn2;
  }
}

// Many query rows (prompt chunks): workgroup (slot x head, row tile of 128 rows),
// 4 waves of 32 rows.  Bound by arithmetic, half of it not matrix products, so
// the codes are turned into 16-bit values once a workgroup: wave w converts keys
// 16w .. 16w + 15 of each 64-key tile into LDS.  LDS holds both operands as their
// 16-byte fragments: K as [column chunk of 8][key], V as [4-key pairs][column][8
// keys], so every fragment is one conflict-free 16-byte read.
// The loop is pipelined so that each stretch between branches holds matrix
// instructions and others that do not wait for them: the scores of tile j + 1
// beside the exponentials of tile j, then the products with V of tile j beside
// the conversion of K of tile j + 2 and V of tile j + 1.
// O^T tile dt, row 16 e + mm is column (D/16) mm + 2 dt + e: the order in which
// code bytes give them.
// 2048 queries of 32 / 8 heads of 128 on 8192 tokens: 240 us, 1.0 PFLOP/s, where a
// large library product of this type reaches 1.2; matrix instructions busy 49 % of
// the cycles, vector ones 59 %, at the 1.8 GHz that the card then runs at (842 us
// by the few-row kernel; 258 us with the same conversion before the stages were
// interleaved).  256 queries on 8448: 53 us, 20 of them before the first and after
// the last tile (three dependent loads, two steps that fill the pipeline, rows out).
constexpr int kRowsTile = 128, kRowsKeys = 64;

template <typename E, int D>
__global__ __launch_bounds__(256, 2) void fa_paged_rows_kernel(PagedAttnArgs a) {
  constexpr int NS = D / 16, ND = D / 32;
  __shared__ u32x4 s_k[2][D / 8][kRowsKeys];
  __shared__ u32x4 s_v[2][kRowsKeys / 8][ND][32];      // [16-key part, h][dt][row]: 4 keys, +8
  __shared__ int s_hole[2][4];
  static_assert(sizeof(s_k) >= 2 * 32 * D * sizeof(float) && sizeof(s_v) >= 2 * 32 * D * sizeof(float),
                "the rows leave through both");
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;              // as a converter
  const int n = lane & 31, hf = lane >> 5;             // as an owner of row n
  const int Hk = a.cache.Hk, hk = blockIdx.x % Hk, slot = blockIdx.x / Hk;
  Chunk ch;
  if (!find_chunk(a, slot, ch)) return;
  const int b = ch.b, rows = a.Sq * a.G;
  const int row0 = (gridDim.y - 1 - blockIdx.y) * kRowsTile;   // the longest sweeps first
  const int count = a.counts ? min(max(scalar_load(a.counts + b), 0), a.Sq) : a.Sq;
  const int base = ch.length - count;

  const int row = row0 + 32 * w + n, qi = row / a.G;
  const int h = hk * a.G + (row - qi * a.G);
  const bool real = row < rows && qi < count;
  const int last = real ? base + qi : -1;
  vec8<E> qf[NS];
  {
    const f16 *qp = a.q + b * a.qs[0] + (int64_t)(real ? qi : 0) * a.qs[1] +
                    (real ? h : 0) * a.qs[2] + 8 * hf;
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      u32x4 raw = *reinterpret_cast<const u32x4 *>(qp + 16 * t);
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j] = real ? raw[j] ^ a.flip : 0u;
      qf[t] = __builtin_bit_cast(vec8<E>, raw);
    }
  }
  const int key0 = ch.index * ch.keys;
  const int i_first = row0 / a.G, i_last = min((row0 + kRowsTile - 1) / a.G, count - 1);
  const int end = i_first < count ? min(min(ch.held, key0 + ch.keys), base + i_last + 1) : 0;
  // this wave's rows see every key below `all` and none from `wend` on
  const int wi = (row0 + 32 * w) / a.G;
  const int all = base + wi + 1;
  const int wend = wi < count ? min(end, base + min((row0 + 32 * w + 31) / a.G, count - 1) + 1) : 0;

  float mx = kLowest, l = 0.0f;
  floatx16 o[ND], s[2];
#pragma unroll
  for (int t = 0; t < ND; ++t) o[t] = floatx16{};

  // Codes in flight, for the next step and the one after it: K of a tile and V of
  // the one before it (whose row is kept until then).
  Tile16<D> raw0, raw1;
  int64_t v_row = 0;
  auto load = [&](int key, Tile16<D> &raw) {
    load_v<D>(a.cache, v_row, m, g, raw);
    v_row = tile_row(a.cache, b, hk, key + 16 * w, end, raw.hole);
    load_k<D>(a.cache, v_row, m, g, raw);
  };
  // pieces of a tile's conversion: K chunk t of this lane's quarter of the
  // columns; columns 2t, 2t + 1 of this lane's V unit
  auto convert_k = [&](int buf, const Tile16<D> &raw, auto T) {
    constexpr int t = decltype(T)::value;
    s_k[buf][ND * g + t][16 * w + m] = fp4_row8<E>(raw_word<D>(raw.k, t), fp4_scale(raw.ks));
    if constexpr (t == 0) s_hole[buf][w] = raw.hole;    // (every lane the same)
  };
  auto convert_v = [&](int buf, const Tile16<D> &raw, auto T) {
    constexpr int t = decltype(T)::value;
    uint32_t x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      x[r] = v_pair<E, D, t>(raw.v, r, fp4_scale((raw.vs >> (8 * r)) & 0xFFu));
    // columns 2t (lo) and 2t + 1 (hi) of keys 4g .. 4g + 3; the halves of the wave
    // swap, so that lanes 0-31 hold 8 keys of the first, 32-63 of the second
    auto x0 = __builtin_amdgcn_permlane32_swap(__builtin_amdgcn_perm(x[1], x[0], 0x05040100u),
                                               __builtin_amdgcn_perm(x[1], x[0], 0x07060302u),
                                               false, false);
    auto x1 = __builtin_amdgcn_permlane32_swap(__builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
                                               __builtin_amdgcn_perm(x[3], x[2], 0x07060302u),
                                               false, false);
    s_v[buf][2 * w + (g & 1)][t][16 * hf + m] = u32x4{x0[0], x1[0], x0[1], x1[1]};
  };
  auto k_frag = [&](int buf, int i) {   // of score instruction i: columns i / 2, keys i % 2
    return __builtin_bit_cast(vec8<E>, s_k[buf][2 * (i >> 1) + hf][32 * (i & 1) + n]);
  };
  auto v_frag = [&](int buf, int i) {   // of V instruction i: keys i / ND, tile i % ND
    return __builtin_bit_cast(vec8<E>, s_v[buf][2 * (i / ND) + hf][i % ND][n]);
  };
  // masks tile `key`'s scores, and moves the running maximum of the rows where they
  // leave the old one behind by 2^8 (of no other row: none depends on its neighbours)
  const int lim = min(last, end - 1);   // the last position that this lane's row sees here
  auto settle = [&](int key, int buf, floatx16 (&x)[2]) {
    if (key + kRowsKeys > all || key + kRowsKeys > end) {
      const int seen = lim - key - 4 * hf;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        x[i >> 4][i & 15] = 32 * (i >> 4) + c_row(i & 15, 0) > seen ? kNegInf : x[i >> 4][i & 15];
    }
    int hole[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) hole[i] = __builtin_amdgcn_readfirstlane(s_hole[buf][i]);
    if (hole[0] | hole[1] | hole[2] | hole[3]) {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i >> 4][i & 15] = hole[i >> 3] ? kNegInf : x[i >> 4][i & 15];
    }
    float top = x[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, x[i >> 4][i & 15]);
    top *= a.c;
    if (__any(top > mx + 8.0f)) {
      float t = max_xor32(top);
      t = t > mx + 8.0f ? t : mx;
      const float f = fast_exp2(mx - t);
      mx = t;
      l *= f;
#pragma unroll
      for (int t2 = 0; t2 < ND; ++t2) o[t2] *= f;
    }
  };

  // Step `key` multiplies tile `key`, takes the scores of the next one, converts K of
  // the one after that and V of the next, and loads what is converted two steps
  // on; two steps before the first tile fill the pipeline.
  auto sweep = [&](int key, Tile16<D> &raw, auto Buf) {
    constexpr int buf = decltype(Buf)::value;
    const bool more = key + kRowsKeys >= key0 && key + kRowsKeys < wend;
    floatx16 next[2];
    next[0] = next[1] = floatx16{};
    if (key >= key0 && key < wend) {
      // The order is fixed here: fragments are read kAhead instructions before
      // the matrix instruction that takes them, and each of those is followed
      // by its share of the other work, which runs beside it.
      constexpr int kAhead = 4, kScore = 2 * NS, kProd = 4 * ND;
      vec8<E> p[4], kf[kScore], vf[kProd];
      static_for<kAhead>([&](auto I) { kf[I] = k_frag(buf ^ 1, I); });
      static_for<kScore>([&](auto I) {
        constexpr int i = decltype(I)::value, per = 32 / kScore;
        if constexpr (i + kAhead < kScore)
          kf[i + kAhead] = k_frag(buf ^ 1, i + kAhead);
        else
          vf[i + kAhead - kScore] = v_frag(buf, i + kAhead - kScore);
        next[i & 1] = mfma32(kf[i], qf[i >> 1], next[i & 1]);
#pragma unroll
        for (int j = per * i; j < per * (i + 1); ++j) {
          const float e = fast_exp2(s[j >> 4][j & 15] * a.c - mx);
          l += e;
          p[j >> 3][j & 7] = (E)e;
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      static_for<kProd>([&](auto I) {
        constexpr int i = decltype(I)::value;
        if constexpr (i + kAhead < kProd) vf[i + kAhead] = v_frag(buf, i + kAhead);
        o[i % ND] = mfma32(vf[i], p[i / ND], o[i % ND]);
        if constexpr (i % 2 == 1 && i < 2 * ND)
          convert_k(buf, raw, std::integral_constant<int, i / 2>{});
        if constexpr (i % 2 == 1 && i >= 2 * ND)
          convert_v(buf ^ 1, raw, std::integral_constant<int, i / 2 - ND>{});
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      if (more) {
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i)
          next[i & 1] = mfma32(k_frag(buf ^ 1, i), qf[i >> 1], next[i & 1]);
      }
      static_for<ND>([&](auto T) { convert_k(buf, raw, T); });
      static_for<ND>([&](auto T) { convert_v(buf ^ 1, raw, T); });
    }
    load(key + 4 * kRowsKeys, raw);
    s[0] = next[0];
    s[1] = next[1];
    if (more) settle(key + kRowsKeys, buf ^ 1, s);
    __syncthreads();
  };
  if (key0 < end) {
    v_row = tile_row(a.cache, b, hk, key0 + 16 * w, end, raw0.hole);
    load_k<D>(a.cache, v_row, m, g, raw0);
    raw0.v = KRaw<D>{};
    raw0.vs = 0;
    load(key0 + kRowsKeys, raw1);
    for (int key = key0 - 2 * kRowsKeys; key < end; key += 2 * kRowsKeys) {
      sweep(key, raw0, std::integral_constant<int, 0>{});
      if (key + kRowsKeys < end) sweep(key + kRowsKeys, raw1, std::integral_constant<int, 1>{});
    }
  }

  leave_count(a, ch, hk);
  // Rows leave through LDS: a lane holds 8 pieces of 2 ND columns of one row, and
  // stores of those would each touch as many lines as lanes (7000 cycles of a
  // workgroup, a third of a short sweep).  Piece mm of row n is kept at mm ^ n % 16.
  l += xor32(l);
  const bool whole = ch.count == 1;
  const bool seen = real && l != 0.0f;                  // (NaN counts as seen)
  const float f = whole ? (seen ? 1.0f / l : 0.0f) : (real ? 1.0f : 0.0f);
  const int64_t part = ((int64_t)(ch.part + ch.index) * Hk + hk) * rows;
  auto leave = [&](auto *kept, auto &&place) {          // kept: 32 rows of this wave in LDS
    typedef std::remove_reference_t<decltype(*kept)> X;
    constexpr int kPiece = 2 * ND;
    typedef X Piece __attribute__((ext_vector_type(kPiece)));
    Piece *mine = reinterpret_cast<Piece *>(kept);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      Piece x;
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        x[2 * t] = (X)(f == 0.0f ? 0.0f : o[t][j] * f);
        x[2 * t + 1] = (X)(f == 0.0f ? 0.0f : o[t][j + 8] * f);
      }
      mine[n * 16 + (c_row(j, hf) ^ (n & 15))] = x;
    }
    // (a wave reads back its own rows: no barrier)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = 64 * j + lane, r = at >> 4, mm = at & 15, out_row = row0 + 32 * w + r;
      if (out_row < rows)
        *reinterpret_cast<Piece *>(place(out_row) + kPiece * mm) = mine[r * 16 + (mm ^ (r & 15))];
    }
  };
  if (whole) {
    leave(reinterpret_cast<E *>(&s_k[0][0][0]) + w * 32 * D, [&](int r) {
      const int i = r / a.G;
      return reinterpret_cast<E *>(a.o) +
             (((int64_t)b * a.Sq + i) * a.H + hk * a.G + (r - i * a.G)) * D;
    });
  } else {                              // two waves' fp32 rows fill s_k, two s_v
    float *half = w < 2 ? reinterpret_cast<float *>(&s_k[0][0][0])
                        : reinterpret_cast<float *>(&s_v[0][0][0][0]);
    leave(half + (w & 1) * 32 * D, [&](int r) { return a.part_o + (part + r) * D; });
  }
  if (hf != 0 || row >= rows) return;
  if (!whole) {
    a.part_ml[(part + row) * 2] = mx;
    a.part_ml[(part + row) * 2 + 1] = real ? l : 0.0f;
  } else if (a.lse) {
    a.lse[((int64_t)b * a.H + h) * a.Sq + qi] = seen ? (mx + fast_log2(l)) * kLn2 : kPosInf;
  }
}

// Joins the chunks of each row of head blockIdx.y of sequence blockIdx.z (rows
// whose sequence is one chunk were written by its workgroup): D / 4 lanes take 4
// columns each of every NS-th chunk of a row, NS such groups a row.  Bound by
// latency (NS = 8, few rows: 3.8 us) or by reading the chunks' rows (NS = 1: 8
// chunks of 8192 rows of 128, 6.9 us, 4.9 TB/s).
template <typename E, int D, int NS, bool ONE>
__global__ __launch_bounds__(256) void fa_paged_merge_kernel(PagedAttnArgs a) {
  constexpr int kLanes = D / 4, kRows = 256 / (kLanes * NS);
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  have(a.lengths, a.part_o, a.part_ml, a.o, a.lse, a.cache.width, a.cache.page_shift, a.cache.Hk,
       a.Sq, a.G, a.H, a.target);
  const int rows = a.Sq * a.G, Hk = a.cache.Hk;
  int count, first = 0;
  if constexpr (ONE) {
    Chunk ch;
    one_sequence(a, ch);
    count = ch.count;
  } else {
    const int *left = chunk_counts(a) + 2 * b;
    count = scalar_load(left);
    first = scalar_load(left + 1);
  }
  if (count == 1) return;
  const int d4 = tid % kLanes, group = tid / kLanes, sub = group % NS;
  const int mine = group / NS, row = blockIdx.x * kRows + mine;
  const bool real = row < rows;
  const int chunks = real ? count : 0;
  float top = kLowest, sum = 0.0f;
  floatx4 acc = {0, 0, 0, 0};
  for (int k0 = sub; k0 < chunks; k0 += 4 * NS) {        // 4 chunks' loads in flight
    float mk[4], lk[4];
    floatx4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = min(k0 + j * NS, count - 1);
      const int64_t p = ((int64_t)(first + k) * Hk + hk) * rows + row;
      const floatx2 ml = *reinterpret_cast<const floatx2 *>(a.part_ml + p * 2);
      mk[j] = ml[0];
      lk[j] = ml[1];
      x[j] = *reinterpret_cast<const floatx4 *>(a.part_o + p * D + 4 * d4);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (k0 + j * NS >= count) break;
      const float t = fmaxf(top, mk[j]), f0 = fast_exp2(top - t), f1 = fast_exp2(mk[j] - t);
      top = t;
      sum = sum * f0 + lk[j] * f1;
      acc = acc * f0 + x[j] * f1;
    }
  }
  if constexpr (NS > 1) {
    __shared__ floatx4 s_acc[kRows][NS][kLanes];
    __shared__ float s_top[kRows][NS], s_sum[kRows][NS];
    s_acc[mine][sub][d4] = acc;
    if (d4 == 0) {
      s_top[mine][sub] = top;
      s_sum[mine][sub] = sum;
    }
    __syncthreads();
    if (sub != 0) return;
    top = s_top[mine][0];
#pragma unroll
    for (int k = 1; k < NS; ++k) top = fmaxf(top, s_top[mine][k]);
    sum = 0.0f;
    acc = floatx4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const float f = fast_exp2(s_top[mine][k] - top);
      sum += s_sum[mine][k] * f;
      acc += s_acc[mine][k][d4] * f;
    }
  }
  if (!real) return;
  const int i = row / a.G, h = hk * a.G + (row - i * a.G);
  E *out = reinterpret_cast<E *>(a.o) + (((int64_t)b * a.Sq + i) * a.H + h) * D;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  vec4<E> v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (E)(acc[j] * inv);
  *reinterpret_cast<vec4<E> *>(out + 4 * d4) = v;
  if (a.lse && d4 == 0)
    a.lse[((int64_t)b * a.H + h) * a.Sq + i] =
        sum == 0.0f ? kPosInf : (top + fast_log2(sum)) * kLn2;
}

}  // namespace fa
