"""The paged 4-bit cache and its attention on the GPU against the float64 oracle.

append / read are exact: a code is the nearest to the 64-bit value, so the values
read back must equal the oracle's.

attend's tolerance, per output: the final rounding, u |o| with u = eps / 2 of
the type; each probability's rounding before the second product, 2^-11 (fp16)
or 2^-16 (two bf16; one, of 8 bits and so 2^-8, with more than 32 rows a
key/value head, whose kernel is bound by arithmetic) of sum p |v|, and once more
for fp16 below 2^-14, 2^-25 of sum |v|; and the scores' errors, which every probability and the sum share in:
a score is off by at most (D + 4) 2^-24 of scale * sum |q k| (fp32 products
and sums) and its exponential by 2^-21 with the sums' own roundings, all twice,
of sum p |v|.  lse: the scores' errors, 2^-21 and 2^-23 of itself.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as orc

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _f64(t):
    return t.detach().cpu().double().numpy()


def _i32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _table(B, width, pages, seed):
    return np.random.default_rng(seed).permutation(pages)[:B * width].reshape(B, width)


def _garbage(cache, seed):
    """Any bytes a freed page can hold: any codes, scales that append writes."""
    g = torch.Generator().manual_seed(seed)
    top = 140 if cache.dtype == F16 else 252
    for name in ("k_codes", "v_codes"):
        t = getattr(cache, name)
        t.copy_(torch.randint(0, 256, t.shape, generator=g).to(torch.uint8))
    for name in ("k_scales", "v_scales"):
        t = getattr(cache, name)
        t.copy_(torch.randint(1, top + 1, t.shape, generator=g).to(torch.uint8))


def _filled(B, lengths, Hk, D, P, dtype, seed, spare=3, width=None, scale=1.0):
    """A cache over garbage with `lengths` tokens stored, its table and model."""
    from flash_attn_volta import PagedKVCache, append_paged
    S = max(max(lengths), 1)
    width = width or -(-S // P)
    pages = B * width + spare
    cache = PagedKVCache(pages, P, Hk, D, dtype)
    _garbage(cache, seed)
    table = _table(B, width, pages, seed)
    k, v = _rand((B, S, Hk, D), dtype, seed + 1, scale), _rand((B, S, Hk, D), dtype, seed + 2, scale)
    model = orc.PagedModel(pages, P, Hk, D, dtype == F16)
    model.store(_f64(k), _f64(v), table, [0] * B, lengths)
    append_paged(cache, k.cuda(), v.cuda(), _i32(table), _i32([0] * B), _i32(lengths))
    return cache, table, model


def _check_attend(out, lse, q, model, table, lengths, counts=None, scale=None):
    dtype, D = out.dtype, out.shape[-1]
    ref, ref_lse, abs_out, abs_v, abs_s = orc.attend(_f64(q), model, table, lengths, counts, scale)
    u = torch.finfo(dtype).eps / 2
    e = 2 * ((D + 4) * 2 ** -24 * abs_s + 2 ** -21)
    many = q.shape[1] * q.shape[2] // model.k.shape[2] > 32
    up, low = ((2 ** -11, 2 ** -25) if dtype == F16 else
               (2 ** -8 if many else 2 ** -16, 2 ** -24))
    tol = (u * np.abs(ref) * 1.01 + (up + e.transpose(0, 2, 1)[..., None]) * abs_out + low * abs_v
           + torch.finfo(dtype).tiny * torch.finfo(dtype).eps)
    err = np.abs(_f64(out) - ref)
    assert (err <= tol).all(), f"out: {np.nanmax(err / tol):.3g} times the tolerance"
    if lse is not None:
        got = _f64(lse)
        assert np.array_equal(np.isinf(got), np.isinf(ref_lse))
        fine = np.isfinite(ref_lse)
        tol = e / 2 + 2 ** -21 + 2 ** -23 * np.abs(ref_lse, where=fine, out=np.zeros_like(ref_lse))
        assert (np.abs(got - ref_lse, where=fine, out=np.zeros_like(got)) <= tol).all()


# -- append and read -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_value_is_stored_as_its_nearest_code(dtype):
    """All 65536 bit patterns, shuffled, and sorted by magnitude (neighbours share
    a block, so every code and border is met)."""
    from flash_attn_volta import PagedKVCache, append_paged, read_paged
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    g = torch.Generator().manual_seed(0)
    x = torch.cat([bits.view(dtype)[torch.randperm(65536, generator=g)],
                   bits.view(dtype)[bits.int().bitwise_and(32767).argsort()]])
    for D in (32, 64, 128):
        v = x.view(1, -1, 1, D)
        S = v.shape[1]
        cache = PagedKVCache(S // 16, 16, 1, D, dtype)
        table = _i32(np.arange(S // 16)[::-1].copy()[None])
        append_paged(cache, v.cuda(), v.cuda().clone(), table, _i32([0]))
        k2, v2 = read_paged(cache, table, _i32([0]), S)
        want = torch.from_numpy(orc.stored(_f64(v), dtype == F16)).to(dtype)
        for name, got in (("k", k2), ("v", v2)):
            assert torch.equal(got.cpu(), want), (name, D, int((got.cpu() != want).sum()))


APPEND = [
    # (B, S, start, counts, Hk, H, D, R, P, interleaved, dtype)
    (1, 1, [0], None, 8, 32, 128, 128, 64, False, BF16),
    (1, 1, [4095], None, 2, 4, 64, 64, 16, False, F16),
    (3, 1, [7, 8, 31], None, 3, 3, 32, 32, 32, False, F16),
    (2, 50, [3, 61], [50, 17], 4, 28, 128, 128, 16, False, BF16),
    (4, 33, [0, 1, 2, 1030], [0, 33, 1, 99], 2, 14, 64, 48, 16, False, F16),
    (1, 200, [13], None, 12, 12, 64, 16, 32, True, F16),
    (2, 9, [5, 100], None, 1, 7, 128, 10, 128, False, BF16),      # unaligned pairs
    (1, 40, [70001], None, 2, 2, 32, 24, 256, False, BF16),       # R / 2 = 12
    (2, 21, [2, 3], [-5, 21], 2, 4, 128, 6, 16, True, F16),
]


@pytest.mark.parametrize("B,S,start,counts,Hk,H,D,R,P,inter,dtype", APPEND)
@pytest.mark.parametrize("layout", ["bshd", "bhsd"])
def test_append_and_read(B, S, start, counts, Hk, H, D, R, P, inter, dtype, layout):
    from flash_attn_volta import (PagedKVCache, RotaryPositions, append_paged, read_paged,
                                  rotary_forward)
    print(f"[case] append {B} {S} {start} {counts} {Hk} {H} {D} {R} {P} {inter} {dtype}", flush=True)
    rot = RotaryPositions(R, base=500000.0, interleaved=inter,
                          scaling={"type": "yarn", "factor": 4, "original_length": 4096})
    width = -(-(max(start) + S) // P)
    pages = B * width + 2
    cache = PagedKVCache(pages, P, Hk, D, dtype)
    _garbage(cache, 5)
    names = ("k_codes", "k_scales", "v_codes", "v_scales")
    before = {n: getattr(cache, n).clone() for n in names}
    table = _table(B, width, pages, 1)
    cpu = [_rand((B, S, h, D), dtype, i) for i, h in enumerate((Hk, Hk, H))]
    k, v, q = ((t.transpose(1, 2).contiguous().cuda().transpose(1, 2) if layout == "bhsd"
                else t.cuda()) for t in cpu)
    cnt = None if counts is None else _i32(counts)
    qo = append_paged(cache, k, v, _i32(table), _i32(start), cnt, q=q, rotary=rot)
    pos = np.asarray(start)[:, None] + np.arange(S)
    assert torch.equal(qo, rotary_forward(q, None, torch.tensor(pos, device="cuda"), rot)[0]) \
        or (qo.float() - rotary_forward(q, None, torch.tensor(pos, device="cuda"), rot)[0].float()
            ).abs().max() <= torch.finfo(dtype).eps * 8          # a rounding border of the angles
    kr = orc.rotate(_f64(cpu[0]), pos, rot.frequencies, rot.attention_factor, inter)
    want_k, want_v = orc.stored(kr, dtype == F16), orc.stored(_f64(cpu[1]), dtype == F16)
    k2, v2 = read_paged(cache, _i32(table), _i32(start), S, cnt)
    n = [S] * B if counts is None else [min(max(c, 0), S) for c in counts]
    for b in range(B):
        assert np.array_equal(_f64(k2)[b, :n[b]], want_k[b, :n[b]])
        assert np.array_equal(_f64(v2)[b, :n[b]], want_v[b, :n[b]])
        assert (k2[b, n[b]:] == 0).all() and (v2[b, n[b]:] == 0).all()
    # every other slot is as it was: put the stored ones back and compare all
    touched = torch.zeros((pages, P), dtype=torch.bool)
    for b in range(B):
        for p in range(start[b], start[b] + n[b]):
            touched[table[b, p // P], p % P] = True
    t = touched.cuda()
    for name in names:
        x, y = getattr(cache, name), before[name]
        if name.startswith("k"):
            same = (x == y).flatten(3).all(-1).all(1)                        # (N, P)
        elif name == "v_codes":                                              # (N,H,P/4,16,4,D/32)
            same = (x == y).permute(0, 2, 4, 1, 3, 5).flatten(3).all(-1).flatten(1)
        else:                                                                # (N,H,P/4,D/32,4)
            same = (x == y).permute(0, 2, 4, 1, 3).flatten(3).all(-1).flatten(1)
        assert bool((same | t).all()), name


def test_append_without_rotation_and_bad_pages():
    """Ids that are no page, positions off the table and before it store nothing,
    and read back as 0."""
    from flash_attn_volta import PagedKVCache, append_paged, read_paged
    Hk, D, P = 2, 64, 16
    cache = PagedKVCache(3, P, Hk, D, F16)
    table = np.array([[1, -1, 2], [2 ** 31 - 1, 0, 3]])
    model = orc.PagedModel(3, P, Hk, D, True)
    k, v = _rand((2, 60, Hk, D), F16, 0), _rand((2, 60, Hk, D), F16, 1)
    start = [-6, 2]
    q = _rand((2, 60, 4, D), F16, 2).cuda()
    out = append_paged(cache, k.cuda(), v.cuda(), _i32(table), _i32(start), q=q)
    assert torch.equal(out, q)                              # no rotation: copied
    model.store(_f64(k), _f64(v), table, start)
    k2, v2 = read_paged(cache, _i32(table), _i32(start), 60)
    for b in range(2):
        rk, rv, _ = model.gather(table, b, range(start[b], start[b] + 60))
        assert np.array_equal(_f64(k2)[b], rk) and np.array_equal(_f64(v2)[b], rv)


def test_pages_past_32_bit_offsets():
    """A pool of more than 2^32 bytes of codes: its last pages."""
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged, read_paged
    Hk, D, P = 8, 128, 256
    pages = 2 ** 32 // (Hk * P * D // 2) + 2
    cache = PagedKVCache(pages, P, Hk, D, BF16)
    assert cache.k_codes.numel() > 2 ** 32
    table = np.array([[pages - 1, 0, pages - 2]])
    k, v = _rand((1, 600, Hk, D), BF16, 0), _rand((1, 600, Hk, D), BF16, 1)
    model = orc.PagedModel(1, P, Hk, D, False)              # (values alone)
    append_paged(cache, k.cuda(), v.cuda(), _i32(table), _i32([0]))
    k2, v2 = read_paged(cache, _i32(table), _i32([0]), 600)
    assert np.array_equal(_f64(k2), orc.stored(_f64(k), False))
    assert np.array_equal(_f64(v2), orc.stored(_f64(v), False))
    model = orc.PagedModel(3, P, Hk, D, False)
    small = np.array([[2, 0, 1]])
    model.store(_f64(k), _f64(v), small, [0])
    q = _rand((1, 2, 16, D), BF16, 3)
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32([600]), return_softmax_lse=True)
    _check_attend(out, lse, q, model, small, [600])


# -- attention -------------------------------------------------------------------------

ATTEND = [
    # (B, Sq, lengths, H, Hk, D, P, dtype)
    (1, 1, [1], 1, 1, 32, 16, F16),
    (1, 1, [4096], 32, 8, 128, 64, BF16),
    (3, 1, [0, 1, 129], 8, 2, 128, 16, F16),
    (5, 1, [5, 300, 17, 1000, 128], 28, 4, 128, 64, BF16),
    (2, 4, [3, 700], 14, 2, 64, 16, F16),              # rows that see nothing
    (2, 3, [257, 90], 4, 4, 32, 32, BF16),
    (1, 2, [513], 64, 8, 128, 128, F16),
    (2, 17, [17, 400], 8, 8, 64, 32, BF16),
    (1, 40, [300], 12, 12, 64, 64, F16),
    (2, 70, [70, 333], 7, 1, 128, 16, BF16),
    (1, 130, [2000], 8, 2, 128, 64, F16),
    (1, 200, [150], 4, 2, 32, 16, F16),                # more queries than tokens
    (1, 1, [2500], 40, 1, 64, 256, BF16),              # 40 rows of one head
]


@pytest.mark.parametrize("B,Sq,lengths,H,Hk,D,P,dtype", ATTEND)
def test_attend(B, Sq, lengths, H, Hk, D, P, dtype):
    from flash_attn_volta import attend_paged
    print(f"[case] attend {B} {Sq} {lengths} {H} {Hk} {D} {P} {dtype}", flush=True)
    cache, table, model = _filled(B, lengths, Hk, D, P, dtype, 11)
    q = _rand((B, Sq, H, D), dtype, 5)
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(lengths), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table, lengths)
    again = attend_paged(q.cuda(), cache, _i32(table), _i32(lengths))
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq,H,Hk,D", [(1, 8, 2, 128), (5, 6, 2, 64), (40, 4, 1, 128), (90, 8, 4, 32)])
def test_attend_padded_batch_holes_strides(dtype, Sq, H, Hk, D):
    """counts, pages that are none, a table wider than the lengths, transposed
    queries, other and negative scales."""
    from flash_attn_volta import attend_paged
    lengths, counts = [200, 47, 3, 0, 130], [Sq, 1, 0, Sq, Sq // 2]
    cache, table, model = _filled(5, lengths, Hk, D, 16, dtype, 3, width=20)
    table[0, 2], table[4, 0], table[1, 0] = -1, 2 ** 30, -2 ** 31
    q = _rand((5, Sq, H, D), dtype, 8)
    qs = q.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    wide = torch.full((5, 23), -7, dtype=torch.int32, device="cuda")
    wide[:, :20] = _i32(table)
    for scale in (None, 0.5, -0.3, 0.0):
        out, lse = attend_paged(qs, cache, wide[:, :20], _i32(lengths), _i32(counts),
                                sm_scale=scale, return_softmax_lse=True)
        _check_attend(out, lse, q, model, table, lengths, counts, scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq,H,Hk,D", [(150, 8, 4, 32), (70, 8, 2, 64), (41, 14, 2, 128)])
def test_attend_many_rows_padded(dtype, Sq, H, Hk, D):
    """As above with more rows than the few-row kernel takes: whole prompt chunks of
    a padded batch, holes, empty rows, all in one chunk (a small table) and
    split (a large one)."""
    from flash_attn_volta import attend_paged
    lengths, counts = [Sq + 300, 47, 3, 0, 130], [Sq, 1, 0, Sq, Sq // 2]
    lengths[4] = 30                                        # fewer tokens than queries
    cache, table, model = _filled(5, lengths, Hk, D, 16, dtype, 3, width=30)
    table[0, 2], table[4, 0], table[1, 0] = -1, 2 ** 30, -2 ** 31
    q = _rand((5, Sq, H, D), dtype, 8)
    for n, cnt in ((lengths, counts), (lengths, None)):
        out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(n),
                                None if cnt is None else _i32(cnt), return_softmax_lse=True)
        _check_attend(out, lse, q, model, table, n, cnt)
    one = attend_paged(q[:1].cuda(), cache, _i32(table[:1]), _i32(lengths[:1]))
    _check_attend(one, None, q[:1], model, table[:1], lengths[:1])


def test_attend_long_prompt_split_and_whole():
    """A prompt against itself, 128-row tiles from one query on to all; many heads
    (one chunk a sequence) and one (split)."""
    from flash_attn_volta import attend_paged
    for B, Sq, H, Hk, D, dtype in ((1, 700, 2, 1, 64, F16), (3, 260, 48, 24, 32, BF16),
                                   (1, 333, 8, 8, 128, BF16)):
        print(f"[case] prompt {B} {Sq} {H} {Hk} {D} {dtype}", flush=True)
        lengths = [Sq] * B
        cache, table, model = _filled(B, lengths, Hk, D, 64, dtype, 2)
        q = _rand((B, Sq, H, D), dtype, 6)
        out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(lengths), return_softmax_lse=True)
        _check_attend(out, lse, q, model, table, lengths)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scores_that_grow_many_rows(dtype):
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged
    L, D, Sq = 900, 128, 300
    cache, table = PagedKVCache(60, 16, 1, D, dtype), _table(1, 57, 60, 0)
    k = _rand((1, L, 1, D), dtype, 0).float()
    k[..., 0] = torch.linspace(-30, 30, L)[None, :, None]
    v = _rand((1, L, 1, D), dtype, 1)
    q = _rand((1, Sq, 1, D), dtype, 2).float()
    q[:, ::2, 0, 0], q[:, 1::2, 0, 0] = 12.0, -12.0
    k, q = k.to(dtype), q.to(dtype)
    model = orc.PagedModel(60, 16, 1, D, dtype == F16)
    model.store(_f64(k), _f64(v), table, [0])
    append_paged(cache, k.cuda(), v.cuda(), _i32(table), _i32([0]))
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32([L]), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table, [L])


def test_a_token_that_is_not_seen_does_not_matter():
    """Later tokens of extreme values, infinities and NaN do not reach earlier
    queries of the same tile: the cache holds finite values, unseen ones weigh 0."""
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged
    for dtype, Sq, H in ((F16, 8, 2), (BF16, 8, 2), (F16, 300, 2), (BF16, 300, 2)):
        L, D = 400, 64
        k, v = _rand((1, L, 1, D), dtype, 0), _rand((1, L, 1, D), dtype, 1)
        k2, v2 = k.clone(), v.clone()
        for t, bad in ((k2, float("inf")), (v2, float("nan"))):
            t[:, -3:] = bad
            t[:, -3:, :, ::2] = torch.finfo(dtype).min
        q = _rand((1, Sq, H, D), dtype, 2).cuda()
        outs = []
        for a, b in ((k, v), (k2, v2)):
            cache, table = PagedKVCache(26, 16, 1, D, dtype), _table(1, 25, 26, 0)
            append_paged(cache, a.cuda(), b.cuda(), _i32(table), _i32([0]))
            outs.append(attend_paged(q, cache, _i32(table), _i32([L])))
        assert torch.equal(outs[0][:, :-3], outs[1][:, :-3])
        assert torch.isfinite(outs[1][:, :-3]).all()


def test_lengths_past_the_table_and_many_sequences():
    from flash_attn_volta import attend_paged
    B = 150                                                # over two scans of 64
    rng = np.random.default_rng(0)
    lengths = [int(x) for x in rng.integers(0, 200, B)]
    cache, table, model = _filled(B, lengths, 1, 32, 16, BF16, 4)
    q = _rand((B, 1, 4, 32), BF16, 8)
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(lengths), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table, lengths)
    full = [table.shape[1] * 16] * B
    cache, table, model = _filled(B, full, 1, 32, 16, BF16, 4)
    over = [n + 5 for n in full]
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(over), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table, over)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq", [1, 50])
def test_scores_that_grow(dtype, Sq):
    """Large, growing scores: the running maximum moves at every step."""
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged
    L, D = 1500, 64
    cache, table = PagedKVCache(100, 16, 1, D, dtype), _table(1, 94, 100, 0)
    k = _rand((1, L, 1, D), dtype, 0).float()
    k[..., 0] = torch.linspace(-30, 30, L)[None, :, None]
    v = _rand((1, L, 1, D), dtype, 1)
    q = _rand((1, Sq, 2, D), dtype, 2).float()
    q[:, :, 0, 0], q[:, :, 1, 0] = 12.0, -12.0
    k, q = k.to(dtype), q.to(dtype)
    model = orc.PagedModel(100, 16, 1, D, dtype == F16)
    model.store(_f64(k), _f64(v), table, [0])
    append_paged(cache, k.cuda(), v.cuda(), _i32(table), _i32([0]))
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32([L]), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table, [L])


# -- a run of them together --------------------------------------------------------------

def test_prompt_then_tokens_as_served():
    """A padded batch of prompts, then single tokens: append with the rotation on
    the way, attend; against the oracle and against the package's dense
    attention over the values read back."""
    from flash_attn_volta import (PagedKVCache, RotaryPositions, append_paged, attend_paged,
                                  flash_attn_forward_gqa, read_paged)
    B, H, Hk, D, P, dtype = 3, 8, 2, 64, 16, BF16
    rot = RotaryPositions(32, base=500000.0, scaling={"type": "linear", "factor": 2})
    cache = PagedKVCache(64, P, Hk, D, dtype)
    _garbage(cache, 0)
    table = _table(B, 8, 64, 2)
    model = orc.PagedModel(64, P, Hk, D, False)
    start, counts = np.zeros(B, dtype=np.int64), [70, 1, 33]
    d_table, d_start = _i32(table), _i32(start)
    for step in range(5):
        S = 70 if step == 0 else 1
        n = counts if step == 0 else [1] * B
        q, k, v = (_rand((B, S, h, D), dtype, 10 * step + i) for i, h in enumerate((H, Hk, Hk)))
        qr = append_paged(cache, k.cuda(), v.cuda(), d_table, d_start, _i32(n), q=q.cuda(),
                          rotary=rot)
        d_start = d_start + _i32(n)
        out, lse = attend_paged(qr, cache, d_table, d_start, _i32(n), return_softmax_lse=True)
        pos = start[:, None] + np.arange(S)
        model.store(orc.rotate(_f64(k), pos, rot.frequencies), _f64(v), table, start, n)
        start = start + n
        _check_attend(out, lse, qr.cpu(), model, table, start, n)
    for b in range(B):                                      # the last step, dense
        kb, vb = read_paged(cache, d_table[b:b + 1], _i32([0]), int(start[b]))
        dense = flash_attn_forward_gqa(qr[b:b + 1], kb, vb, causal=True)
        assert (dense.float() - out[b:b + 1].float()).abs().max() <= 2 ** -6


def test_a_captured_step_follows_its_inputs():
    """One decode step in a graph: replays read the lengths, the table and the
    tokens that the buffers hold then, and two graphs and eager calls keep
    apart."""
    from flash_attn_volta import (PagedKVCache, RotaryPositions, append_paged, attend_paged,
                                  release_workspaces)
    B, H, Hk, D, P, dtype = 4, 16, 4, 128, 64, F16
    rot = RotaryPositions(D)
    caches = [PagedKVCache(40, P, Hk, D, dtype) for _ in range(3)]
    table = _i32(_table(B, 10, 40, 2))
    q, k, v = (_rand((B, 1, h, D), dtype, i).cuda() for i, h in enumerate((H, Hk, Hk)))
    held = _i32([0, 100, 500, 639])
    for c in caches:
        kk, vv = _rand((B, 639, Hk, D), dtype, 7).cuda(), _rand((B, 639, Hk, D), dtype, 8).cuda()
        append_paged(c, kk, vv, table, _i32([0] * B), held)

    def step(cache):
        qr = append_paged(cache, k, v, table, held, q=q, rotary=rot)
        return attend_paged(qr, cache, table, held + 1, return_softmax_lse=True)

    step(caches[2])
    torch.cuda.synchronize()
    graphs = []
    for c in caches[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step(c)))
            # (a second call in the same capture)
            attend_paged(q, c, table, held)
    release_workspaces()
    for rep in range(4):
        for t, s in ((q, 50), (k, 60), (v, 70)):
            t.copy_(_rand(t.shape, dtype, s + rep).cuda())
        if rep == 2:
            held.copy_(_i32([638, 0, 1, 77]))
        want = step(caches[2])
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), rep


def test_calls_on_two_streams():
    from flash_attn_volta import attend_paged
    cache, table, model = _filled(4, [900, 33, 5, 400], 4, 128, 64, BF16, 1)
    q = _rand((4, 1, 16, 128), BF16, 2).cuda()
    t, n = _i32(table), _i32([900, 33, 5, 400])
    want = attend_paged(q, cache, t, n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(attend_paged(q, cache, t, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_empty_and_refused():
    from flash_attn_volta import (PagedKVCache, RotaryPositions, append_paged, attend_paged,
                                  read_paged)
    from flash_attn_volta.forward import FlashAttnArgumentError
    c = PagedKVCache(4, 16, 2, 64, F16)
    t, n = _i32([[0, 1]]), _i32([3])
    k = torch.zeros((1, 5, 2, 64), dtype=F16, device="cuda")
    q = torch.zeros((1, 5, 4, 64), dtype=F16, device="cuda")
    assert append_paged(c, k[:, :0], k[:, :0], t, n) is None
    assert append_paged(c, k[:0], k[:0], t[:0], n[:0], q=q[:0]).shape == (0, 5, 4, 64)
    assert append_paged(c, k, k, t, n, q=q[:, :, :0]).shape == (1, 5, 0, 64)
    assert attend_paged(q[:, :0], c, t, n).shape == (1, 0, 4, 64)
    assert read_paged(c, t, n, 0)[0].shape == (1, 0, 2, 64)
    rot = RotaryPositions(128)
    for bad in (lambda: append_paged(c, k.bfloat16(), k, t, n), lambda: append_paged(c, k, k, t.long(), n),
                lambda: append_paged(c, k, k[:, :4], t, n), lambda: append_paged(c, k[:, :, :1], k, t, n),
                lambda: append_paged(c, k, k, t, n.long()), lambda: append_paged(c, k, k, t, None),
                lambda: append_paged(c, k, k, t, n, _i32([1, 2])),
                lambda: append_paged(c, k, k, t, n, rotary=rot),
                lambda: append_paged(c, k, k, t, n, q=q[:, :3]),
                lambda: append_paged(c, k, k, t[:, :0], n), lambda: append_paged(c, k.cpu(), k, t, n),
                lambda: attend_paged(q[:, :, :3], c, t, n), lambda: attend_paged(q, c, t, n.cpu()),
                lambda: attend_paged(q, None, t, n), lambda: attend_paged(q[0], c, t, n),
                lambda: attend_paged(q, c, t, n, sm_scale=float("nan")),
                lambda: read_paged(c, t, n, -1), lambda: read_paged(c, t[0], n, 1),
                lambda: PagedKVCache(4, 24, 2, 64), lambda: PagedKVCache(4, 16, 2, 96),
                lambda: PagedKVCache(0, 16, 2, 64), lambda: PagedKVCache(4, 8, 2, 64),
                lambda: PagedKVCache.from_tensors(c.k_codes, c.k_scales, c.v_codes, c.k_scales, F16),
                lambda: PagedKVCache.from_tensors(c.k_codes, c.k_scales, c.v_codes, c.v_scales,
                                                  torch.float32)):
        with pytest.raises((FlashAttnArgumentError, RuntimeError)):
            bad()


def test_other_layouts_are_taken():
    """Tables, lengths and rows that the kernels do not read in place are copied:
    strided tables, misaligned rows, strides that are no multiple of 8."""
    from flash_attn_volta import (PagedKVCache, RotaryPositions, append_paged, attend_paged,
                                  read_paged, rotary_forward)
    B, S, H, Hk, D, P = 2, 5, 4, 2, 64, 16
    rot = RotaryPositions(32)
    q, k, v = (_rand((B, S, h, D), F16, i).cuda() for i, h in enumerate((H, Hk, Hk)))
    table, start, n = _i32([[3, 0], [1, 2]]), _i32([9, 14]), _i32([14, 19])
    pos = torch.arange(S, device="cuda")

    def run(q, k, v, table, start, n):
        cache = PagedKVCache(4, P, Hk, D, F16)
        qo = append_paged(cache, k, v, table, start, q=q, rotary=rot)
        return (qo, *read_paged(cache, table, start, S), attend_paged(qo, cache, table, n),
                rotary_forward(q, k, pos, rot)[1])

    def shifted(t):                       # 2 bytes off 16-byte alignment
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    def odd(t):                           # rows 4 elements apart from the next head's
        wide = torch.zeros((*t.shape[:2], t.shape[2] * (D + 4)), dtype=t.dtype, device="cuda")
        view = wide.view(*t.shape[:3], D + 4)[..., :D]
        view.copy_(t)
        return view

    want = run(q, k, v, table, start, n)
    twice = lambda t: torch.stack((t, t), dim=-1).flatten(-2)[..., ::2]  # noqa: E731
    for args in ((shifted(q), shifted(k), shifted(v), table, start, n),
                 (odd(q), odd(k), odd(v), table.t().contiguous().t(), start, n),
                 (q, k, v, twice(table), twice(start), twice(n))):
        assert all(torch.equal(a, b) for a, b in zip(run(*args), want))


def test_the_python_way_gives_the_same(monkeypatch):
    """Without the C++ module every call goes through Python."""
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged, paged, read_paged
    lengths = [700, 33]
    outs = []
    for cpp in (paged._cpp, None):
        monkeypatch.setattr(paged, "_cpp", cpp)
        cache, table, model = _filled(2, lengths, 2, 64, 16, BF16, 7)
        q = _rand((2, 3, 8, 64), BF16, 1).cuda()
        out, lse = attend_paged(q, cache, _i32(table), _i32(lengths), return_softmax_lse=True)
        k, v = read_paged(cache, _i32(table), _i32([1, 2]), 40, _i32([40, 3]))
        outs.append((out, lse, k, v, append_paged(cache, k[:, :1], v[:, :1], _i32(table),
                                                  _i32([0, 0]), q=q[:, :1])))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_shared_pages_and_one_table_for_all():
    """Sequences that share a prefix's pages, and one table row for every sequence."""
    from flash_attn_volta import attend_paged
    cache, table, model = _filled(1, [100], 2, 64, 16, F16, 9)
    q = _rand((3, 2, 4, 64), F16, 1)
    lengths = [100, 37, 2]
    shared = _i32(table).expand(3, -1)
    out, lse = attend_paged(q.cuda(), cache, shared, _i32(lengths), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table.repeat(3, 0), lengths)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq,H,Hk,D", [(1, 8, 2, 128), (5, 6, 2, 64), (3, 4, 4, 32), (40, 4, 1, 128),
                                       (150, 8, 4, 32), (70, 16, 2, 64), (41, 14, 2, 128)])
def test_attend_split_padded(dtype, Sq, H, Hk, D):
    """Tables large enough that long sequences are split and joined, beside short,
    empty and padded ones: counts, holes, early rows that see nothing."""
    from flash_attn_volta import attend_paged
    lengths, counts = [1500, 47, 3, 0, 130, 700], [Sq, 1, 0, Sq, Sq // 2, Sq]
    cache, table, model = _filled(6, lengths, Hk, D, 16, dtype, 3, width=130)
    table[0, 2], table[0, 60], table[4, 0], table[5, 43] = -1, -7, 2 ** 30, 6 * 130 + 3
    q = _rand((6, Sq, H, D), dtype, 8)
    for cnt in (counts, None):
        out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(lengths),
                                None if cnt is None else _i32(cnt), return_softmax_lse=True)
        _check_attend(out, lse, q, model, table, lengths, cnt)


@pytest.mark.parametrize("B,seed", [(63, 0), (64, 1), (65, 2), (130, 3)])
def test_split_many_sequences(B, seed):
    """More sequences than a wave counts at once, some of many chunks."""
    from flash_attn_volta import attend_paged
    rng = np.random.default_rng(seed)
    lengths = [int(x) for x in rng.integers(0, 300, B)]
    for i, n in ((0, 2600), (B // 2, 1900), (B - 1, 2570)):
        lengths[i] = n
    cache, table, model = _filled(B, lengths, 1, 32, 16, BF16, 4, width=165)
    q = _rand((B, 1, 4, 32), BF16, 8)
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(lengths), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table, lengths)


@pytest.mark.parametrize("H,Hk,D,dtype", [(24, 12, 64, F16), (8, 8, 128, BF16), (4, 2, 32, BF16)])
def test_prompt_in_pieces(H, Hk, D, dtype):
    """A 1300-token prompt in pieces of odd sizes gives each row what it gets in one."""
    from flash_attn_volta import attend_paged
    L = 1300
    cache, table, model = _filled(1, [L], Hk, D, 64, dtype, 2)
    q = _rand((1, L, H, D), dtype, 6).cuda()
    whole = attend_paged(q, cache, _i32(table), _i32([L]))
    at = 0
    # a probability and an output are rounded, half a step each, and twice: two calls
    tol = 4 * 4 * torch.finfo(dtype).eps / 2
    for n in (1, 2, 13, 64, 65, 300, 511, 344):
        piece = attend_paged(q[:, at:at + n], cache, _i32(table), _i32([at + n]))
        diff = (piece.float() - whole[:, at:at + n].float()).abs().max()
        assert diff <= tol * whole[:, at:at + n].float().abs().max(), (at, n, float(diff))
        at += n
    assert at == L


@pytest.mark.parametrize("Sq,H,L", [(5, 2, 400), (8, 8, 400), (300, 2, 900), (40, 2, 2100)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_row_does_not_depend_on_its_neighbours(dtype, Sq, H, L):
    """Bit for bit: queries with scores far larger, in rows of the same tiles, move
    no other row's running maximum."""
    from flash_attn_volta import attend_paged
    cache, table, _ = _filled(1, [L], 1, 64, 16, dtype, 5)
    q = _rand((1, Sq, H, 64), dtype, 7)
    loud = q.clone()
    loud[:, 1::2] *= 40
    a, b = (attend_paged(x.cuda(), cache, _i32(table), _i32([L])) for x in (q, loud))
    assert torch.equal(a[:, ::2], b[:, ::2])
    assert not torch.equal(a[:, 1::2], b[:, 1::2])


def test_counts_below_zero_are_none():
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged, read_paged
    low = -2 ** 31
    cache, table = PagedKVCache(4, 16, 2, 32, BF16), _i32([[0, 1]])
    k, v, q = (_rand((1, 24, 2, 32), BF16, i).cuda() for i in range(3))
    for n in (low, low + 5, -1):
        append_paged(cache, k, v, table, _i32([3]), _i32([n]))
        assert not any(getattr(cache, t).any() for t in ("k_codes", "k_scales", "v_codes", "v_scales"))
    append_paged(cache, k, v, table, _i32([0]))
    for n in (low, -1):
        assert not any(t.any() for t in read_paged(cache, table, _i32([0]), 24, _i32([n])))
        out, lse = attend_paged(q, cache, table, _i32([24]), _i32([n]), return_softmax_lse=True)
        assert not out.any() and torch.isinf(lse).all()
        assert not attend_paged(q, cache, table, _i32([n])).any()


def test_a_batch_of_over_2_31_keys():
    """Sequences that share one page hold 2^30 keys each, of which no query is asked;
    the one beside them keeps its result.  (Over 1024 heads: no sequence is split.)"""
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged
    P, H, L = 4096, 1025, 100
    cache = PagedKVCache(1, P, H, 32, BF16)
    k, v, q = (_rand((1, n, H, 32), BF16, i).cuda() for i, n in enumerate((L, L, 1)))
    one = torch.zeros((1, 2 ** 30 // P), dtype=torch.int32, device="cuda")
    append_paged(cache, k, v, one, _i32([0]))
    alone = attend_paged(q, cache, one, _i32([L]))
    assert alone.any()
    for at in range(3):
        lengths, counts = [2 ** 30] * 3, [0] * 3
        lengths[at], counts[at] = L, 1
        out = attend_paged(q.expand(3, -1, -1, -1), cache, one.expand(3, -1), _i32(lengths),
                           _i32(counts))
        assert torch.equal(out[at], alone[0])
        assert not out[[i for i in range(3) if i != at]].any()


def test_calls_inside_a_compiled_function():
    """Traced functions call them between the pieces of their graphs."""
    from flash_attn_volta import (PagedKVCache, RotaryPositions, append_paged,
                                  apply_rotary_positions, attend_paged, read_paged)
    rotary, pos = RotaryPositions(64), torch.arange(5, device="cuda")[None]
    q, k = (_rand((2, 5, h, 64), F16, h).cuda().requires_grad_() for h in (8, 2))
    table, start = _i32(np.arange(8).reshape(2, 4)), _i32([0, 3])

    def train(q, k):
        a, b = apply_rotary_positions(q * 2, k, pos, rotary)
        return (a * b.repeat_interleave(4, 2)).float().sum()

    def serve(q, k, cache):
        rotated = append_paged(cache, k, k + 1, table, start, q=q, rotary=rotary)
        out, lse = attend_paged(rotated * 1, cache, table, start + 5, return_softmax_lse=True)
        return (out * 1, lse, *read_paged(cache, table, start, 5))

    grads, results = [], []
    for wrap in (lambda f: f, lambda f: torch.compile(f, backend="eager")):
        grads.append(torch.autograd.grad(wrap(train)(q, k), (q, k)))
        with torch.no_grad():
            results.append(wrap(serve)(q, k, PagedKVCache(8, 16, 2, 64, F16)))
    for a, b in (*zip(*grads), *zip(*results)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B,Sq,Hk", [(255, 1, 1), (256, 4, 2), (257, 1, 1), (515, 1, 1), (300, 140, 1)])
def test_split_hundreds_of_sequences(B, Sq, Hk):
    """As test_split_many_sequences, with more sequences and rows; and the same batch in
    a table that is not split."""
    from flash_attn_volta import attend_paged
    rng = np.random.default_rng(B)
    lengths = [int(x) for x in rng.integers(0, 150, B)]
    for i, n in ((1, 2100), (B // 2, 0), (B - 1, 2111)):
        lengths[i] = n
    cache, table, model = _filled(B, lengths, Hk, 32, 16, F16, 4, width=132)
    q = _rand((B, Sq, Hk, 32), F16, 8)
    out, lse = attend_paged(q.cuda(), cache, _i32(table), _i32(lengths), return_softmax_lse=True)
    _check_attend(out, lse, q, model, table, lengths)
    short = [min(n, 500) for n in lengths]
    out, lse = attend_paged(q.cuda(), cache, _i32(table[:, :32]), _i32(short),
                            return_softmax_lse=True)
    _check_attend(out, lse, q, model, table[:, :32], short)


def test_a_batch_of_over_2_32_keys_that_may_be_split():
    """As test_a_batch_of_over_2_31_keys, with chunks in reach: 512 heads, two a round."""
    from flash_attn_volta import PagedKVCache, append_paged, attend_paged
    P, H, L, B = 4096, 512, 100, 6
    cache = PagedKVCache(1, P, H, 32, F16)
    k, v, q = (_rand((1, n, H, 32), F16, i).cuda() for i, n in enumerate((L, L, 1)))
    one = torch.zeros((1, 2 ** 30 // P), dtype=torch.int32, device="cuda")
    append_paged(cache, k, v, one, _i32([0]))
    alone = attend_paged(q, cache, one[:, :1], _i32([L]))
    assert alone.any()
    for at in (0, 3, 5):
        lengths, counts = [2 ** 30] * B, [0] * B
        lengths[at], counts[at] = L, 1
        out = attend_paged(q.expand(B, -1, -1, -1), cache, one.expand(B, -1), _i32(lengths),
                           _i32(counts))
        assert torch.equal(out[at], alone[0])
        assert not out[[i for i in range(B) if i != at]].any()


@pytest.mark.parametrize("B,Sq", [(1, 1), (5, 3), (70, 1), (3, 100)])
def test_replays_split_as_their_lengths_say(B, Sq):
    """One captured call serves batches of any lengths: many chunks, one, none."""
    from flash_attn_volta import attend_paged
    most = 2600
    cache, table, model = _filled(B, [most] * B, 2, 64, 16, F16, 4, width=170)
    q, t, lengths = _rand((B, Sq, 4, 64), F16, 8).cuda(), _i32(table), _i32([most] * B)
    attend_paged(q, cache, t, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = attend_paged(q, cache, t, lengths, return_softmax_lse=True)
    rng = np.random.default_rng(B)
    for now in ([0] * B, [most] * B, [most] + [1] * (B - 1), rng.integers(0, 200, B),
                rng.integers(0, most, B), [100] * B):
        lengths.copy_(_i32(now))
        want, want_lse = attend_paged(q, cache, t, lengths, return_softmax_lse=True)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    _check_attend(out, lse, q, model, table, [100] * B)
