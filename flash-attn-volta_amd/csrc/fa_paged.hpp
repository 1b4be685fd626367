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
  int units, unit_shift;                 // of a row of q (rotary_units)
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
// tokens.
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
    for (int i = tid; i < nt * r2; i += kAppendThreads) {
      const int t = i / r2, j = i - t * r2;
      cs[t * slots + pair_slot(j, r2)] =
          rotary_cos_sin<float>(start + i0 + t, a.rot.steps[j], (float)a.rot.factor);
    }
    if (r2) __syncthreads();
    const int u = tid & ((1 << a.unit_shift) - 1), lanes = kAppendThreads >> a.unit_shift;
    if (u >= a.units) return;
    const int step = lanes * (gridDim.y - a.parts), dt = step / a.H, dh = step - dt * a.H;
    int t = (blockIdx.y - a.parts) * lanes + (tid >> a.unit_shift), h = t % a.H;
    t /= a.H;
    for (; t < nt; t += dt, h += dh) {
      if (h >= a.H) {
        h -= a.H;
        if (++t >= nt) break;
      }
      rotate_unit<E>(a.q + b * a.qs[0] + (int64_t)(i0 + t) * a.qs[1] + h * a.qs[2],
                     a.q_out + b * a.qos[0] + (int64_t)(i0 + t) * a.qos[1] + h * a.qos[2], u,
                     cs + t * slots, r2, a.rot.interleaved != 0);
    }
    return;
  }
  if (a.counts) nt = min(nt, a.counts[b] - i0);
  if (nt <= 0) return;
  CosSin<double> *cs = reinterpret_cast<CosSin<double> *>(smem);
  for (int i = tid; i < nt * r2; i += kAppendThreads) {
    const int t = i / r2, j = i - t * r2;
    cs[t * slots + pair_slot(j, r2)] =
        rotary_cos_sin<double>(start + i0 + t, a.rot.steps[j], a.rot.factor);
  }
  if (r2) __syncthreads();
  const int Hk = a.cache.Hk;
  // whole blocks of 32 columns stay together: nt * Hk * NCH is a multiple of 4
  for (int i = blockIdx.y * kAppendThreads + tid; i < nt * Hk * NCH; i += a.parts * kAppendThreads) {
    const int c = i % NCH, th = i / NCH, h = th / nt, t = th - h * nt;
    const int64_t pos = start + i0 + t;
    const int page = page_of(a.cache, b, pos);
    const int slot = (int)(pos & ((1 << a.cache.page_shift) - 1));
    const f16 *kr = a.k + b * a.ks[0] + (int64_t)(i0 + t) * a.ks[1] + h * a.ks[2];
    const f16 *vr = a.v + b * a.vs[0] + (int64_t)(i0 + t) * a.vs[1] + h * a.vs[2];
    float vy[8], ky[8];
    load8<E, float>(vr + 8 * c, vy);
    if (r2) {
      double y[8];
      rotate8<E, double>(kr, c, cs + t * slots, r2, a.rot.interleaved != 0, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) ky[j] = odd_float(y[j]);
    } else {
      load8<E, float>(kr + 8 * c, ky);
    }
    unsigned kb, vb;
    const uint32_t kw = quantise8(ky, a.top, a.max_byte, kb);
    const uint32_t vw = quantise8(vy, a.top, a.max_byte, vb);
    if (page < 0) continue;
    const int64_t row = paged_row(a.cache, page, h, slot);
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
// (behind counts[b], outside the table, on a page that is none).
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
  float *part_o;                        // (slots, Hk, rows, D) unnormalised
  float *part_ml;                       // (slots, Hk, rows, 2): maximum (log2), sum
  int B, Sq, H, G;
  int slots;                            // chunks in all, at most
  int target;                           // chunks aimed at
  float c;                              // |sm_scale| log2 e
  uint32_t flip;                        // sign bits xor-ed into q (negative scale)
};

// Queries of a packed tile: row n of (b, hk) is query n / G of head hk G + n % G.
// Keys a row sees: positions <= lengths - counts + query.
constexpr int kUnit = 128;              // keys: one step of the 4 waves
constexpr float kLowest = -3.4028234663852886e38f;

struct Chunk {
  int b, index, count, keys;            // `count` chunks of `keys` keys in sequence b
  int first;                            // slot of the sequence's chunk 0
};

__device__ __forceinline__ int held_keys(const PagedAttnArgs &a, int b) {
  const int64_t cap = (int64_t)a.cache.width << a.cache.page_shift;
  return (int)max((int64_t)0, min((int64_t)a.lengths[b], cap));
}

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// Splits all sequences' keys evenly: chunks of the same whole number of units
// (the last of a sequence shorter), about `target` of them, whatever the lengths.  The
// host knows no lengths; every wave counts them for itself (B loads) and finds
// the sequence of its slot; one that holds nothing is a chunk too, which writes
// its zeros.  target + B slots cover every chunk, B with a target of 1 (then no
// sequence is split).  With
// `by_sequence` the argument is a sequence and its chunks are returned.
__device__ __forceinline__ bool find_chunk(const PagedAttnArgs &a, int want, bool by_sequence,
                                           Chunk &out) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    total += b < a.B ? (held_keys(a, b) + kUnit - 1) / kUnit : 0;
  }
  total = wave_sum(total);
  const int units = max(1, (total + a.target - 1) / a.target);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    const int u = b < a.B ? (held_keys(a, b) + kUnit - 1) / kUnit : 0;
    const int n = b < a.B ? max(1, (u + units - 1) / units) : 0;
    int upto = n;                       // inclusive prefix sum
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(upto, m, 64);
      if (lane >= m) upto += o;
    }
    const int first = before + upto - n;
    const bool mine = by_sequence ? b == want : (want >= first && want < first + n);
    const uint64_t hit = __ballot(mine);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      out.b = __builtin_amdgcn_readfirstlane(b0 + src);
      out.first = __builtin_amdgcn_readfirstlane(__shfl(first, src, 64));
      out.count = __builtin_amdgcn_readfirstlane(__shfl(n, src, 64));
      out.index = want - out.first;
      out.keys = __builtin_amdgcn_readfirstlane(units) * kUnit;
      return true;
    }
    before += __shfl(upto, 63, 64);
  }
  return false;
}

template <int D> struct KRaw { u32x4 w; };
template <> struct KRaw<64> { u32x2 w; };
template <> struct KRaw<32> { uint32_t w; };

template <int D> __device__ __forceinline__ uint32_t raw_word(const KRaw<D> &r, int i) { return r.w[i]; }
template <> __device__ __forceinline__ uint32_t raw_word<32>(const KRaw<32> &r, int) { return r.w; }

// One wave's share of a 16-key tile: codes of key m's quarter g of the columns,
// of V group g's unit m, and their scales.
template <int D> struct Tile16 {
  KRaw<D> k, v;
  uint32_t ks, vs;
  bool hole;
};

template <int D>
__device__ __forceinline__ void load_tile(const PagedCache &c, int b, int hk, int key, int end,
                                          int m, int g, Tile16<D> &t) {
  // (a page that is none: page 0 is read instead, its keys masked)
  int page = key < end ? page_of(c, b, key) : -1;
  page = __builtin_amdgcn_readfirstlane(page);
  t.hole = page < 0;
  const int64_t row = paged_row(c, max(page, 0), hk, key & ((1 << c.page_shift) - 1));
  const uint8_t *kc = c.k_codes + row * (D / 2), *ksc = c.k_scales + row * (D / 32);
  const uint8_t *vc = c.v_codes + row * (D / 2), *vsc = c.v_scales + row * (D / 32);
  t.k = *reinterpret_cast<const KRaw<D> *>(kc + m * (D / 2) + g * (D / 8));
  t.v = *reinterpret_cast<const KRaw<D> *>(vc + (g * 16 + m) * (D / 8));
  t.ks = ksc[m * (D / 32) + g * D / 128];
  t.vs = *reinterpret_cast<const uint32_t *>(vsc + (g * (D / 32) + m * D / 512) * 4);
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
template <typename E, int D, int NT>
__global__ __launch_bounds__(256) void fa_paged_few_kernel(PagedAttnArgs a) {
  constexpr int KS = D / 32, ND = D / 16, NW = 4;
  constexpr int PARTS = std::is_same<E, bf16>::value ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = a.cache.Hk, hk = blockIdx.x % Hk, slot = blockIdx.x / Hk;
  Chunk ch;
  if (!find_chunk(a, slot, false, ch)) return;
  const int b = ch.b, rows = a.Sq * a.G, row0 = blockIdx.y * (16 * NT);
  const int held = held_keys(a, b);
  const int count = a.counts ? min(max(a.counts[b], 0), a.Sq) : a.Sq;
  const int base = a.lengths[b] - count;          // position of query 0

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
      // a new maximum only where the old one is left behind by 2^8
      if (__any(top > mx[nt] + 8.0f)) {
        float t = fmaxf(top, __shfl_xor(top, 16, 64));
        t = fmaxf(t, xor32(t));
        t = fmaxf(t, mx[nt]);
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
  __shared__ float s_o[NW][D][17];                // 17: columns of a row in different banks
  __shared__ float s_m[NW][16], s_l[NW][16];
  const int64_t part = ((int64_t)slot * Hk + hk) * rows;
  const bool whole = ch.count == 1;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float ls = l[nt] + __shfl_xor(l[nt], 16, 64);
    ls += xor32(ls);
    if (g == 0) {
      s_m[w][m] = mx[nt];
      s_l[w][m] = ls;
    }
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s_o[w][ND * (4 * g + i) + t][m] = o[nt][t][i];
    __syncthreads();
    for (int e = tid; e < 16 * D; e += 64 * NW) {
      const int d = e % D, n = e / D, row = row0 + 16 * nt + n;
      if (row < rows) {
        float top = s_m[0][n];
#pragma unroll
        for (int k = 1; k < NW; ++k) top = fmaxf(top, s_m[k][n]);
        const int i = row / a.G, h = hk * a.G + (row - i * a.G);
        float sum = 0.0f, acc = 0.0f;
        if (i < count) {
#pragma unroll
          for (int k = 0; k < NW; ++k) {
            const float f = fast_exp2(s_m[k][n] - top);
            sum += s_l[k][n] * f;
            acc += s_o[k][d][n] * f;
          }
        }
        if (whole) {
          reinterpret_cast<E *>(a.o)[(((int64_t)b * a.Sq + i) * a.H + h) * D + d] =
              (E)(sum > 0.0f ? acc / sum : (sum == 0.0f ? 0.0f : sum));
          if (a.lse && d == 0)
            a.lse[((int64_t)b * a.H + h) * a.Sq + i] =
                sum == 0.0f ? kPosInf : (top + fast_log2(sum)) * kLn2;
        } else {
          a.part_o[(part + row) * D + d] = acc;
          if (d == 0) {
            a.part_ml[(part + row) * 2] = top;
            a.part_ml[(part + row) * 2 + 1] = sum;
          }
        }
      }
    }
    __syncthreads();
  }
}

// Many query rows (prompt chunks): workgroup (slot x head, row tile of 128 rows),
// 4 waves of 32 rows.  Bound by arithmetic, half of it not matrix products, so
// the codes are turned into 16-bit values once a workgroup: wave w converts keys
// 16w .. 16w + 15 of each 64-key tile into LDS, one tile ahead of the products
// and with the next tile's codes in flight.  LDS holds both operands as their
// 16-byte fragments: K as [column chunk of 8][key], V as [4-key pairs][column][8
// keys], so every fragment is one conflict-free 16-byte read.
// O^T tile dt, row rr is column (D/16)(rr / 2) + 2 dt + rr % 2: the order in
// which code bytes give them.
constexpr int kRowsTile = 128, kRowsKeys = 64;

template <typename E, int D>
__global__ __launch_bounds__(256, 2) void fa_paged_rows_kernel(PagedAttnArgs a) {
  constexpr int NS = D / 16, ND = D / 32;
  __shared__ u32x4 s_k[2][D / 8][kRowsKeys];
  __shared__ u32x2 s_v[2][kRowsKeys / 8][ND][32][2];   // [16-key part, h][dt][rr][4 keys, +8]
  __shared__ int s_hole[2][4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;              // as a converter
  const int n = lane & 31, hf = lane >> 5;             // as an owner of row n
  const int Hk = a.cache.Hk, hk = blockIdx.x % Hk, slot = blockIdx.x / Hk;
  Chunk ch;
  if (!find_chunk(a, slot, false, ch)) return;
  const int b = ch.b, rows = a.Sq * a.G;
  const int row0 = (gridDim.y - 1 - blockIdx.y) * kRowsTile;   // the longest sweeps first
  const int held = held_keys(a, b);
  const int count = a.counts ? min(max(a.counts[b], 0), a.Sq) : a.Sq;
  const int base = a.lengths[b] - count;

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
  const int end = i_first < count ? min(min(held, key0 + ch.keys), base + i_last + 1) : 0;
  // this wave's rows see every key below `all` and none from `wend` on
  const int wi = (row0 + 32 * w) / a.G;
  const int all = base + wi + 1;
  const int wend = wi < count ? min(end, base + min((row0 + 32 * w + 31) / a.G, count - 1) + 1) : 0;

  float mx = kLowest, l = 0.0f;
  floatx16 o[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) o[t] = floatx16{};

  Tile16<D> raw;
  auto load = [&](int key) { load_tile<D>(a.cache, b, hk, key + 16 * w, end, m, g, raw); };
  auto convert = [&](int buf) {
    const float sc = fp4_scale(raw.ks);
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
      s_k[buf][(D / 32) * g + t][16 * w + m] = fp4_row8<E>(raw_word<D>(raw.k, t), sc);
    float vs[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) vs[r] = fp4_scale((raw.vs >> (8 * r)) & 0xFFu);
    auto columns = [&](auto S) {
      constexpr int s = decltype(S)::value;
      uint32_t x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = v_pair<E, D, s>(raw.v, r, vs[r]);
      u32x2 *to = &s_v[buf][2 * w + (g & 1)][s][2 * m][g >> 1];
      to[0] = u32x2{__builtin_amdgcn_perm(x[1], x[0], 0x05040100u),
                    __builtin_amdgcn_perm(x[3], x[2], 0x05040100u)};
      to[2] = u32x2{__builtin_amdgcn_perm(x[1], x[0], 0x07060302u),
                    __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
    };
    columns(std::integral_constant<int, 0>{});
    if constexpr (ND > 1) columns(std::integral_constant<int, 1>{});
    if constexpr (ND > 2) {
      columns(std::integral_constant<int, 2>{});
      columns(std::integral_constant<int, 3>{});
    }
    if (lane == 0) s_hole[buf][w] = raw.hole;
  };

  if (key0 < end) {
    load(key0);
    convert(0);
    if (key0 + kRowsKeys < end) load(key0 + kRowsKeys);
  }
  __syncthreads();
  int buf = 0;
  for (int key = key0; key < end; key += kRowsKeys) {
    if (key + kRowsKeys < end) {
      convert(buf ^ 1);
      if (key + 2 * kRowsKeys < end) load(key + 2 * kRowsKeys);
    }
    if (key < wend) {
      floatx16 s[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        s[kt] = floatx16{};
#pragma unroll
        for (int t = 0; t < NS; ++t)
          s[kt] = mfma32(__builtin_bit_cast(vec8<E>, s_k[buf][2 * t + hf][32 * kt + n]), qf[t], s[kt]);
      }
      const bool holes = s_hole[buf][0] | s_hole[buf][1] | s_hole[buf][2] | s_hole[buf][3];
      if (key + kRowsKeys > all || key + kRowsKeys > end || __builtin_amdgcn_readfirstlane(holes)) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int kk = key + 32 * kt + c_row(i, hf);
            if (kk > last || kk >= end || s_hole[buf][2 * kt + i / 8]) s[kt][i] = kNegInf;
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
      top *= a.c;
      // a new maximum only where the old one is left behind by 2^8
      if (__any(top > mx + 8.0f)) {
        const float t = fmaxf(max_xor32(top), mx);
        const float f = fast_exp2(mx - t);
        mx = t;
        l *= f;
#pragma unroll
        for (int t2 = 0; t2 < ND; ++t2) o[t2] *= f;
      }
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          vec8<E> p;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float e = fast_exp2(s[kt][8 * u + i] * a.c - mx);
            l += e;
            p[i] = (E)e;
          }
#pragma unroll
          for (int t = 0; t < ND; ++t)
            o[t] = mfma32(*reinterpret_cast<const vec8<E> *>(&s_v[buf][4 * kt + 2 * u + hf][t][n][0]),
                          p, o[t]);
        }
    }
    __syncthreads();
    buf ^= 1;
  }

  if (row >= rows) return;
  l += xor32(l);
  const bool seen = real && l != 0.0f;                  // (NaN counts as seen)
  const bool whole = ch.count == 1;
  const float f = whole ? (seen ? 1.0f / l : 0.0f) : (real ? 1.0f : 0.0f);
  const int64_t part = ((int64_t)slot * Hk + hk) * rows + row;
  E *out = reinterpret_cast<E *>(a.o) + (((int64_t)b * a.Sq + qi) * a.H + h) * D;
  // registers 2j, 2j + 1 of every dt are 2 ND consecutive columns
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int d = NS * (c_row(2 * j, hf) / 2);
    float x[2 * ND];
#pragma unroll
    for (int t = 0; t < ND; ++t) {
      x[2 * t] = seen || !whole ? o[t][2 * j] * f : 0.0f;
      x[2 * t + 1] = seen || !whole ? o[t][2 * j + 1] * f : 0.0f;
    }
    if (whole) {
      E y[2 * ND];
#pragma unroll
      for (int t = 0; t < 2 * ND; ++t) y[t] = (E)x[t];
      __builtin_memcpy(__builtin_assume_aligned(out + d, 4 * ND), y, sizeof y);
    } else {
      __builtin_memcpy(__builtin_assume_aligned(a.part_o + part * D + d, 8 * ND), x, sizeof x);
    }
  }
  if (hf != 0) return;
  if (!whole) {
    a.part_ml[part * 2] = mx;
    a.part_ml[part * 2 + 1] = real ? l : 0.0f;
  } else if (a.lse) {
    a.lse[((int64_t)b * a.H + h) * a.Sq + qi] = seen ? (mx + fast_log2(l)) * kLn2 : kPosInf;
  }
}

// Joins the chunks of row blockIdx.x of head blockIdx.y of sequence blockIdx.z
// (rows whose sequence is one chunk were written by its workgroup).
template <typename E, int D>
__global__ __launch_bounds__(256) void fa_paged_merge_kernel(PagedAttnArgs a) {
  const int row = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int rows = a.Sq * a.G, Hk = a.cache.Hk;
  Chunk ch;
  find_chunk(a, b, true, ch);
  const int i = row / a.G, h = hk * a.G + (row - i * a.G);
  E *out = reinterpret_cast<E *>(a.o) + (((int64_t)b * a.Sq + i) * a.H + h) * D;
  if (ch.count == 1) return;
  constexpr int NS = 256 / (D / 4);               // chunks at a time, D / 4 lanes each
  const int d4 = tid % (D / 4), sub = tid / (D / 4);
  float top = kLowest, sum = 0.0f;
  floatx4 acc = {0, 0, 0, 0};
  for (int k = sub; k < ch.count; k += NS) {
    const int64_t p = ((int64_t)(ch.first + k) * Hk + hk) * rows + row;
    const float mk = a.part_ml[p * 2], lk = a.part_ml[p * 2 + 1];
    const floatx4 x = *reinterpret_cast<const floatx4 *>(a.part_o + p * D + 4 * d4);
    const float t = fmaxf(top, mk), f0 = fast_exp2(top - t), f1 = fast_exp2(mk - t);
    top = t;
    sum = sum * f0 + lk * f1;
    acc = acc * f0 + x * f1;
  }
  __shared__ floatx4 s_acc[NS][D / 4];
  __shared__ float s_top[NS], s_sum[NS];
  s_acc[sub][d4] = acc;
  if (d4 == 0) {
    s_top[sub] = top;
    s_sum[sub] = sum;
  }
  __syncthreads();
  if (tid >= D / 4) return;
  top = s_top[0];
#pragma unroll
  for (int k = 1; k < NS; ++k) top = fmaxf(top, s_top[k]);
  sum = 0.0f;
  acc = floatx4{0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    const float f = fast_exp2(s_top[k] - top);
    sum += s_sum[k] * f;
    acc += s_acc[k][tid] * f;
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  vec4<E> v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (E)(acc[j] * inv);
  *reinterpret_cast<vec4<E> *>(out + 4 * tid) = v;
  if (a.lse && tid == 0)
    a.lse[((int64_t)b * a.H + h) * a.Sq + i] =
        sum == 0.0f ? kPosInf : (top + fast_log2(sum)) * kLn2;
}

}  // namespace fa
