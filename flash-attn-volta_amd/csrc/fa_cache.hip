// fa_cache.hip -- C ABI of the rotary positions, the paged 4-bit cache and the
// attention over it (include/fa_mi355x.h): argument checks, launch shapes and
// launches.  Checks run before any HIP call.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "fa_mi355x.h"
#include "fa_paged.hpp"
#include "fa_rotary.hpp"

namespace {

using fa::bf16;
using fa::f16;

bool aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_dtype(int dtype) {
  return dtype == FA_DTYPE_F16 || dtype == FA_DTYPE_BF16 ? FA_OK : FA_ERR_DTYPE;
}

// A (B, S, heads, D) tensor of 16-bit rows read or written 16 bytes at a time;
// every offset is 64-bit in these kernels.  An output's rows must not overlap.
int check_rows(const void *p, const int64_t *st, int B, int S, int heads, int D, bool output) {
  if (p == nullptr || st == nullptr) return FA_ERR_NULL_POINTER;
  if (!aligned(p, 16)) return FA_ERR_ALIGNMENT;
  if (st[3] != 1) return FA_ERR_STRIDE;
  const int64_t n[3] = {B, S, heads};
  double span = D;
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0 || (st[i] & 7) != 0) return FA_ERR_STRIDE;
    span += (double)(n[i] - 1) * st[i];
  }
  if (span > 4.0e18) return FA_ERR_TOO_LARGE;
  if (!output) return FA_OK;
  // in order of stride, each stride at least the extent of what is nested in it
  int64_t extent = D;
  bool used[3] = {false, false, false};
  for (int k = 0; k < 3; ++k) {
    int at = -1;
    for (int i = 0; i < 3; ++i)
      if (!used[i] && n[i] > 1 && (at < 0 || st[i] < st[at])) at = i;
    if (at < 0) break;
    used[at] = true;
    if (st[at] < extent) return FA_ERR_STRIDE;
    extent += st[at] * (n[at] - 1);
  }
  return FA_OK;
}

void copy3(int64_t *to, const int64_t *st) {
  for (int i = 0; i < 3; ++i) to[i] = st[i];
}

constexpr int64_t kMaxThreads = 0xFFFFF000;   // of a grid dimension

int launch_status() { return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH; }

// Compute units of the device `stream` belongs to (the current device for
// NULL), cached per device.
int stream_cus(hipStream_t stream) {
  static std::atomic<int> cache[64];
  int dev = -1;
  if (stream == nullptr || hipStreamGetDevice(stream, &dev) != hipSuccess || dev < 0) {
    (void)hipGetLastError();
    if (hipGetDevice(&dev) != hipSuccess) {
      (void)hipGetLastError();
      return 256;
    }
  }
  if (dev >= 64) return 256;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) {
      (void)hipGetLastError();
      n = 256;
    }
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// -- rotary ----------------------------------------------------------------------

int check_rotary(const int64_t *steps, double factor, int rotary_dim, int D) {
  if (steps == nullptr) return FA_ERR_NULL_POINTER;
  if (!aligned(steps, 8)) return FA_ERR_ALIGNMENT;
  if (rotary_dim < 2 || rotary_dim > D || (rotary_dim & 1)) return FA_ERR_HEAD_DIM;
  return isfinite((float)factor) ? FA_OK : FA_ERR_SCALE;   // (q is rotated in fp32)
}

int log2_up(int n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}

template <typename E>
int launch_rotary(fa::RotaryArgs a, int D, hipStream_t st) {
  a.D = D;
  a.unit_shift = log2_up(fa::rotary_units(D));
  // One token to a workgroup, its heads over several, until the workgroups
  // fill the GPU; then 4, whose angles are one each for the 256 lanes at
  // R = 128, or 8 of at most 128 units, which would leave lanes without work
  // (8 x 1001 tokens, 24 heads of 64: 14.5 / 12.7 us with 4 / 8; 4096, 40 of 128:
  // 17.5 / 21.4).
  const int cus = stream_cus(st);
  const int64_t rows = (int64_t)a.heads[0] + a.heads[1], lanes = fa::kRotaryThreads >> a.unit_shift;
  const size_t lds = fa::pair_slots(a.rot.r2) * sizeof(fa::CosSin<float>);
  if (a.tokens < 4 * cus) {
    int64_t y = 4 * cus / a.tokens;
    const int64_t most = (rows + lanes - 1) / lanes;
    y = y > most ? most : (y < 1 ? 1 : y);
    fa::fa_rotary_kernel<E, 1>
        <<<dim3((unsigned)a.tokens, (unsigned)y), fa::kRotaryThreads, lds, st>>>(a);
  } else if (rows << a.unit_shift <= 128) {
    fa::fa_rotary_kernel<E, 8>
        <<<dim3((unsigned)((a.tokens + 7) / 8)), fa::kRotaryThreads, 8 * lds, st>>>(a);
  } else {
    fa::fa_rotary_kernel<E, 4>
        <<<dim3((unsigned)((a.tokens + 3) / 4)), fa::kRotaryThreads, 4 * lds, st>>>(a);
  }
  return launch_status();
}

// -- cache -----------------------------------------------------------------------

int check_cache(const fa_paged_cache *c, const int32_t *table, int64_t table_stride, int B, int D,
                int dtype) {
  if (c == nullptr || c->k_codes == nullptr || c->k_scales == nullptr || c->v_codes == nullptr ||
      c->v_scales == nullptr || table == nullptr)
    return FA_ERR_NULL_POINTER;
  if (int rc = check_dtype(dtype)) return rc;
  if (D != 32 && D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (B <= 0 || c->pages <= 0 || c->heads <= 0 || c->width <= 0) return FA_ERR_SHAPE;
  if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) != 0) return FA_ERR_SHAPE;
  if (table_stride < 0) return FA_ERR_STRIDE;
  if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scales, 4) ||
      !aligned(c->v_scales, 4) || !aligned(table, 4))
    return FA_ERR_ALIGNMENT;
  // positions and counts of 128-key units are 32-bit, z grids 16-bit
  if ((double)c->width * c->page_size > (double)(1 << 30)) return FA_ERR_TOO_LARGE;
  if ((double)c->width * c->page_size / 128 * B > (double)(1 << 30)) return FA_ERR_TOO_LARGE;
  if ((double)c->pages * c->heads * c->page_size * D > 4.0e18) return FA_ERR_TOO_LARGE;
  if (B > 65535 || c->heads > 65535) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

fa::PagedCache device_cache(const fa_paged_cache *c, const int32_t *table, int64_t table_stride) {
  return fa::PagedCache{static_cast<uint8_t *>(c->k_codes), static_cast<uint8_t *>(c->k_scales),
                        static_cast<uint8_t *>(c->v_codes), static_cast<uint8_t *>(c->v_scales),
                        table, table_stride, c->pages, c->width,
                        __builtin_ctz((unsigned)c->page_size), c->heads};
}

template <typename E, int D>
int launch_append(const fa::AppendArgs &a, dim3 grid, hipStream_t st) {
  const size_t lds = a.rot.steps ? fa::kAppendTokens * fa::pair_slots(a.rot.r2) *
                                       sizeof(fa::CosSin<double>)
                                 : 0;
  fa::fa_paged_append_kernel<E, D><<<grid, fa::kAppendThreads, lds, st>>>(a);
  return launch_status();
}

template <typename E>
int launch_append_d(const fa::AppendArgs &a, int D, dim3 grid, hipStream_t st) {
  return D == 128 ? launch_append<E, 128>(a, grid, st)
         : D == 64 ? launch_append<E, 64>(a, grid, st)
                   : launch_append<E, 32>(a, grid, st);
}

template <typename E, int D>
int launch_read(const fa::ReadArgs &a, hipStream_t st) {
  fa::fa_paged_read_kernel<E, D><<<(unsigned)((a.work + 255) / 256), 256, 0, st>>>(a);
  return launch_status();
}

template <typename E>
int launch_read_d(const fa::ReadArgs &a, int D, hipStream_t st) {
  return D == 128 ? launch_read<E, 128>(a, st)
         : D == 64 ? launch_read<E, 64>(a, st)
                   : launch_read<E, 32>(a, st);
}

// -- attention -------------------------------------------------------------------

// The launch of these sizes: the kernel (`nt` column tiles of 16 rows a
// workgroup, 0: the one for many rows), row tiles, chunks aimed at (for each
// head and row tile) and at most.
struct AttnPlan {
  int nt, row_tiles, target, slots;
  int64_t rows;
  // partial results of the chunks of split sequences (fa::find_chunk): 68 MiB at
  // most on 256 compute units
  size_t o_bytes(int Hk, int D) const {
    return target > 1 ? (size_t)(target + 1) * Hk * rows * D * sizeof(float) : 0;
  }
  size_t bytes(int B, int Hk, int D) const {
    return target > 1 ? o_bytes(Hk, D) + (size_t)(target + 1) * Hk * rows * 2 * sizeof(float) +
                            (B > 1 ? (size_t)B * 2 * sizeof(int) : 0)
                      : 0;
  }
};

AttnPlan attn_plan(int B, int Sq, int H, int Hk, int D, int cus, int64_t capacity) {
  AttnPlan p;
  p.rows = (int64_t)Sq * (H / Hk);
  // The many-row kernel pays from 65 rows on, from 257 where a call has at most
  // 8192 in all and is bound by latency (us with the join, few rows / many: 64 rows
  // of 32 x 8 heads on 2000 tokens 41 / 55; 128 of 64 heads on 4000 42 / 43; 192 of 64
  // 66 / 52; 256 of 128 on 2000 73 / 59; 128, 256 of 8 heads on 8000 23 / 33, 29 / 35;
  // 128 of 32 on 4000 29 / 35).
  const bool few = p.rows <= 64 || (p.rows <= 256 && p.rows * Hk * B <= 8192);
  p.nt = p.rows <= 16 ? 1 : (few ? 2 : 0);
  const int tile = p.nt ? 16 * p.nt : fa::kRowsTile;
  p.row_tiles = (int)((p.rows + tile - 1) / tile);
  // As many chunks as workgroups are resident at once: a second, short round
  // costs more than the longer sweeps.  The few-row kernel has 4 a compute unit
  // (2 with two column tiles: 16 x 4 queries of 14 / 2 heads of 64 on up to 5000
  // tokens 8.9 us, 11.4 with 4), the many-row one 2.
  const int64_t resident = (int64_t)(p.nt == 1 ? 4 : 2) * cus / ((int64_t)Hk * p.row_tiles);
  // Where a table holds few positions no sequence is split: the join costs more than
  // the sweeps, whose steps take longer with wider rows and two tiles (us, split /
  // whole: one query of 32 / 8 heads of 128 on 1024 tokens 9.3 / 9.0, on 1280 9.5 /
  // 10.5; of 14 / 2 of 64 on 1280 9.3 / 8.2, on 1536 9.3 / 9.2, on 2048 9.4 / 11.3; 8
  // queries of 32 / 8 of 128 on 512 9.5 / 8.9, on 768 9.6 / 10.9; 16 of 14 / 2 of 64 on
  // 1024 9.7 / 8.9).  With a workgroup for each compute unit anyway: 32 x 1 of 32 / 8 of
  // 128 on 2048 19.0 / 16.0, on up to 2048 14.9 / 15.1, on up to 2560 16.5 / 18.2; 64 x
  // 8 of 14 / 2 of 64 on up to 2048 17.5 / 14.4.  Many rows: 256 of 32 / 8 of 128 on
  // 1024 30.6 / 25.5, on 1280 29.1 / 30.3; 4 x 128 of 14 / 2 of 64 on 1024 20.4 / 19.7.
  const int wide = D * p.nt;
  const bool every_cu = p.nt != 0 && (int64_t)B * Hk * p.row_tiles >= cus;
  const int64_t enough = p.nt == 0   ? 1024
                         : every_cu  ? 2048
                         : wide > 128 ? 640
                         : wide > 64  ? 1024
                                      : 1408;
  p.target = resident < 1 || capacity <= enough ? 1 : (int)resident;
  p.slots = p.target > 1 ? std::max(p.target, (p.target + 1) / 2 + B) : B;   // fa::find_chunk
  // (no more than the units that the table holds)
  const int64_t units = (std::min(capacity, (int64_t)1 << 30) + fa::kUnit - 1) / fa::kUnit;
  p.slots = (int)std::min((int64_t)p.slots, units * B);
  return p;
}

int check_attn_sizes(int B, int Sq, int H, int Hk, int D, int dtype) {
  if (int rc = check_dtype(dtype)) return rc;
  if (B <= 0 || Sq <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0) return FA_ERR_SHAPE;
  if (D != 32 && D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (B > 65535 || Hk > 65535 || (int64_t)Sq * (H / Hk) > (1 << 20)) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

template <typename E, int D>
int launch_attn(const fa::PagedAttnArgs &a, const AttnPlan &p, hipStream_t st) {
  const dim3 grid((unsigned)(p.slots * a.cache.Hk), (unsigned)p.row_tiles);
  if (p.nt == 1)
    fa::fa_paged_few_kernel<E, D, 1><<<grid, 256, 0, st>>>(a);
  else if (p.nt == 2)
    fa::fa_paged_few_kernel<E, D, 2><<<grid, 256, 0, st>>>(a);
  else
    fa::fa_paged_rows_kernel<E, D><<<grid, 256, 0, st>>>(a);
  if (int rc = launch_status()) return rc;
  if (p.target == 1) return FA_OK;
  // Groups of D / 4 lanes that share a row's chunks: 8, or one where rows alone
  // fill the GPU (256 queries of 32 heads of 128, 8 chunks: 9.4 / 6.4 us).
  constexpr int kGroups = 1024 / D;
  auto blocks = [&](int ns) {
    const int64_t each = kGroups / ns;
    return dim3((unsigned)((p.rows + each - 1) / each), (unsigned)a.cache.Hk, (unsigned)a.B);
  };
  const bool many = p.rows * a.cache.Hk * a.B >= (int64_t)4 * kGroups * stream_cus(st);
  const auto merge = a.B == 1 ? (many ? fa::fa_paged_merge_kernel<E, D, 1, true>
                                      : fa::fa_paged_merge_kernel<E, D, 8, true>)
                              : (many ? fa::fa_paged_merge_kernel<E, D, 1, false>
                                      : fa::fa_paged_merge_kernel<E, D, 8, false>);
  merge<<<blocks(many ? 1 : 8), 256, 0, st>>>(a);
  return launch_status();
}

template <typename E>
int launch_attn_d(const fa::PagedAttnArgs &a, const AttnPlan &p, int D, hipStream_t st) {
  return D == 128 ? launch_attn<E, 128>(a, p, st)
         : D == 64 ? launch_attn<E, 64>(a, p, st)
                   : launch_attn<E, 32>(a, p, st);
}

}  // namespace

extern "C" {

int fa_rotary(const void *q, const void *k, void *q_out, void *k_out, const int64_t *steps,
              double factor, int rotary_dim, int flags, const void *positions,
              const int64_t position_strides[2], int B, int S, int H, int Hk, int D,
              const int64_t q_strides[4], const int64_t k_strides[4],
              const int64_t q_out_strides[4], const int64_t k_out_strides[4], int dtype,
              void *stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (B <= 0 || S <= 0 || H <= 0 || Hk < 0) return FA_ERR_SHAPE;
  if (D < 8 || D > 256 || (D & 7)) return FA_ERR_HEAD_DIM;
  if (int rc = check_rotary(steps, factor, rotary_dim, D)) return rc;
  if (positions == nullptr || position_strides == nullptr) return FA_ERR_NULL_POINTER;
  if (!aligned(positions, (flags & FA_ROTARY_POS64) ? 8 : 4)) return FA_ERR_ALIGNMENT;
  if (position_strides[0] < 0 || position_strides[1] < 0) return FA_ERR_STRIDE;
  if (int rc = check_rows(q, q_strides, B, S, H, D, false)) return rc;
  if (int rc = check_rows(q_out, q_out_strides, B, S, H, D, true)) return rc;
  if (Hk > 0) {
    if (int rc = check_rows(k, k_strides, B, S, Hk, D, false)) return rc;
    if (int rc = check_rows(k_out, k_out_strides, B, S, Hk, D, true)) return rc;
  }
  const int64_t tokens = (int64_t)B * S;
  // a grid has under 2^32 threads: 64 a token; rows are counted in 32 bits
  if (tokens > kMaxThreads / 64 || ((int64_t)H + Hk) * (D / 8) > (1 << 24)) return FA_ERR_TOO_LARGE;
  fa::RotaryArgs a{};
  a.x[0] = static_cast<const f16 *>(q);
  a.y[0] = static_cast<f16 *>(q_out);
  copy3(a.xs[0], q_strides);
  copy3(a.ys[0], q_out_strides);
  if (Hk > 0) {
    a.x[1] = static_cast<const f16 *>(k);
    a.y[1] = static_cast<f16 *>(k_out);
    copy3(a.xs[1], k_strides);
    copy3(a.ys[1], k_out_strides);
  }
  a.heads[0] = H;
  a.heads[1] = Hk;
  a.rot = fa::RotaryTable{steps, factor, rotary_dim / 2, (flags & FA_ROTARY_INTERLEAVED) != 0,
                          (flags & FA_ROTARY_INVERSE) != 0};
  a.positions = positions;
  a.pb = position_strides[0];
  a.ps = position_strides[1];
  a.pos64 = (flags & FA_ROTARY_POS64) != 0;
  a.S = S;
  a.tokens = tokens;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == FA_DTYPE_F16 ? launch_rotary<f16>(a, D, st) : launch_rotary<bf16>(a, D, st);
}

int fa_paged_append(const fa_paged_cache *cache, const int32_t *table, int64_t table_stride,
                    const void *k, const void *v, const void *q, void *q_out,
                    const int32_t *start, const int32_t *counts, const int64_t *steps,
                    double factor, int rotary_dim, int flags, int B, int S, int H, int D,
                    const int64_t k_strides[4], const int64_t v_strides[4],
                    const int64_t q_strides[4], const int64_t q_out_strides[4], int dtype,
                    void *stream) {
  if (int rc = check_cache(cache, table, table_stride, B, D, dtype)) return rc;
  if (S <= 0) return FA_ERR_SHAPE;
  if (start == nullptr) return FA_ERR_NULL_POINTER;
  if (!aligned(start, 4) || !aligned(counts, 4)) return FA_ERR_ALIGNMENT;
  if (steps != nullptr)
    if (int rc = check_rotary(steps, factor, rotary_dim, D)) return rc;
  if (int rc = check_rows(k, k_strides, B, S, cache->heads, D, false)) return rc;
  if (int rc = check_rows(v, v_strides, B, S, cache->heads, D, false)) return rc;
  if (q != nullptr) {
    if (H <= 0) return FA_ERR_SHAPE;
    if (int rc = check_rows(q, q_strides, B, S, H, D, false)) return rc;
    if (int rc = check_rows(q_out, q_out_strides, B, S, H, D, true)) return rc;
  }
  if ((int64_t)(q ? H : 0) > (1 << 20) || S > (1 << 26)) return FA_ERR_TOO_LARGE;
  fa::AppendArgs a{};
  a.cache = device_cache(cache, table, table_stride);
  a.k = static_cast<const f16 *>(k);
  a.v = static_cast<const f16 *>(v);
  copy3(a.ks, k_strides);
  copy3(a.vs, v_strides);
  if (q != nullptr) {
    a.q = static_cast<const f16 *>(q);
    a.q_out = static_cast<f16 *>(q_out);
    copy3(a.qs, q_strides);
    copy3(a.qos, q_out_strides);
    a.H = H;
  }
  a.start = start;
  a.counts = counts;
  if (steps != nullptr)
    a.rot = fa::RotaryTable{steps, factor, rotary_dim / 2, (flags & FA_ROTARY_INTERLEAVED) != 0, 0};
  a.S = S;
  // fp16 caches hold up to 6 * 2^13, what their type can hold
  a.top = dtype == FA_DTYPE_F16 ? 65504.0f : 3.3895313892515355e38f;
  a.max_byte = dtype == FA_DTYPE_F16 ? 127 + 13 : 127 + 125;
  const int64_t tiles = ((int64_t)S + 14) / 8;
  // Parts of a tile: a lane does up to 4 chunks of keys and values, or units of
  // q, where the grid fills the GPU without more parts, down to one where not.
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t tok = S < fa::kAppendTokens ? S : fa::kAppendTokens;
  const int64_t kv = tok * cache->heads * (D / 8);
  int64_t qu = 0;
  if (q != nullptr) {
    a.unit_shift = log2_up(fa::rotary_units(D));
    qu = tok * H << a.unit_shift;
  }
  int64_t each = 4 * fa::kAppendThreads;
  while (each > fa::kAppendThreads && (kv + qu) / each * tiles * B < 2 * stream_cus(st)) each /= 2;
  auto parts = [&](int64_t n) { return n > 64 * each ? 64 : (n + each - 1) / each; };
  a.parts = (int)parts(kv);
  const dim3 grid((unsigned)tiles, (unsigned)(a.parts + parts(qu)), (unsigned)B);
  return dtype == FA_DTYPE_F16 ? launch_append_d<f16>(a, D, grid, st)
                               : launch_append_d<bf16>(a, D, grid, st);
}

int fa_paged_read(const fa_paged_cache *cache, const int32_t *table, int64_t table_stride, void *k,
                  void *v, const int32_t *start, const int32_t *counts, int B, int n, int D,
                  int dtype, void *stream) {
  if (int rc = check_cache(cache, table, table_stride, B, D, dtype)) return rc;
  if (n <= 0) return FA_ERR_SHAPE;
  if (k == nullptr || v == nullptr || start == nullptr) return FA_ERR_NULL_POINTER;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(start, 4) || !aligned(counts, 4))
    return FA_ERR_ALIGNMENT;
  const double work = (double)B * n * cache->heads * (D / 8);
  if (work > (double)kMaxThreads) return FA_ERR_TOO_LARGE;
  const fa::ReadArgs a{device_cache(cache, table, table_stride), static_cast<f16 *>(k),
                       static_cast<f16 *>(v), start, counts, n,
                       (int64_t)B * n * cache->heads * (D / 8)};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == FA_DTYPE_F16 ? launch_read_d<f16>(a, D, st) : launch_read_d<bf16>(a, D, st);
}

size_t fa_paged_attn_workspace_bytes(int B, int Sq, int H, int Hk, int D) {
  if (check_attn_sizes(B, Sq, H, Hk, D, FA_DTYPE_F16) != FA_OK) return 0;
  return attn_plan(B, Sq, H, Hk, D, stream_cus(nullptr), INT64_MAX).bytes(B, Hk, D);
}

int fa_paged_attn(const void *q, const fa_paged_cache *cache, const int32_t *table,
                  int64_t table_stride, const int32_t *lengths, const int32_t *counts, void *o,
                  float *lse, void *workspace, size_t workspace_bytes, int B, int Sq, int H, int D,
                  const int64_t q_strides[4], float sm_scale, int dtype, void *stream) {
  if (int rc = check_cache(cache, table, table_stride, B, D, dtype)) return rc;
  if (int rc = check_attn_sizes(B, Sq, H, cache->heads, D, dtype)) return rc;
  if (lengths == nullptr || o == nullptr) return FA_ERR_NULL_POINTER;
  if (!aligned(o, 16) || !aligned(lengths, 4) || !aligned(counts, 4) || !aligned(lse, 4))
    return FA_ERR_ALIGNMENT;
  if (int rc = check_rows(q, q_strides, B, Sq, H, D, false)) return rc;
  if (!isfinite(sm_scale)) return FA_ERR_SCALE;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int Hk = cache->heads;
  // (the size does not depend on the cache: a small one may leave it unused)
  const int cus = stream_cus(st);
  const AttnPlan most = attn_plan(B, Sq, H, Hk, D, cus, INT64_MAX);
  if ((int64_t)most.slots * Hk > kMaxThreads / 256) return FA_ERR_TOO_LARGE;
  if (most.bytes(B, Hk, D) > 0) {
    if (workspace == nullptr || workspace_bytes < most.bytes(B, Hk, D)) return FA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return FA_ERR_ALIGNMENT;
  }
  const AttnPlan p = attn_plan(B, Sq, H, Hk, D, cus, (int64_t)cache->width * cache->page_size);
  fa::PagedAttnArgs a{};
  a.cache = device_cache(cache, table, table_stride);
  a.q = static_cast<const f16 *>(q);
  copy3(a.qs, q_strides);
  a.o = static_cast<f16 *>(o);
  a.lse = lse;
  a.lengths = lengths;
  a.counts = counts;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float *>(static_cast<char *>(workspace) + p.o_bytes(Hk, D));
  a.B = B;
  a.Sq = Sq;
  a.H = H;
  a.G = H / Hk;
  a.target = p.target;
  // never 0, so that masked (-inf) scores stay -inf
  a.c = fmaxf(fabsf(sm_scale) * fa::kLog2e, 1e-30f);
  a.flip = sm_scale < 0 ? 0x80008000u : 0u;
  return dtype == FA_DTYPE_F16 ? launch_attn_d<f16>(a, p, D, st) : launch_attn_d<bf16>(a, p, D, st);
}

}  // extern "C"
