"""The serving-step operators (paged K/V cache write, read and attention; logit
rules with the greedy choice) against plain definitions in 64 bits.

Tolerances come from the roundings that the operators name, not from runs:
  * cache codes and scales are the format's own f32 steps: exact;
  * attention: the output's rounding u |o|; each weight's rounding to f16 and, in
    an 8-bit cache, each value's, 2^-11 each of A = sum p |v| (2^-21 for f32
    queries, whose weights keep 22 bits); f32 sums of n keys, n 2^-23 A; and the
    scores: q to 2^-15 of its largest number (2^-21 for f32 queries), f32 sums of
    the dims, d 2^-23, which move each weight by at most twice that; and f16's
    smallest steps: 2^-32 of the largest |v| for each key's weight (held as 2^7 p),
    2^-25 for an f16 output;
  * logits: see test_logits.
"""
import ctypes
import math

import numpy as np
import pytest

from malaga_b200 import _lib

gpu_only = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(request):
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from malaga_b200 import ops as o

    return o


def _torch():
    import torch

    return torch


# ---------------------------------------------------------------------------
# Plain definitions

def q8_plain(x):
    """Codes and scales of rows x [..., dim] (numpy f32): the format's f32 steps."""
    x = x.astype(np.float32)
    finite = np.isfinite(x).all(-1)
    top = np.abs(np.where(np.isfinite(x), x, 0)).max(-1).astype(np.float32)
    d = (top / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        q = (x / d[..., None]).astype(np.float32)
    code = np.where((d > 0)[..., None] & finite[..., None], np.clip(np.rint(np.nan_to_num(q)), -127, 127), 0)
    return code.astype(np.int8), np.where(finite, d, np.float32(np.nan))


class Case:
    """A cache with stale contents everywhere, sequences over shuffled pages, and their plain values."""

    def __init__(self, ops, fmt, heads, dim, page, new, lens, seed=0, spare=2, stale=math.nan):
        torch = _torch()
        rng = np.random.default_rng(seed)
        self.fmt, self.heads, self.dim, self.page, self.new, self.lens = fmt, heads, dim, page, new, lens
        need = [-(-c // page) for c in lens]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.tables, at = [], 0
        for n in need:
            self.tables.append([int(p) for p in order[at: at + n]])
            at += n
        self.cache = ops.PagedKV.empty(pages, heads, page, dim, fmt)
        self.values = []  # per sequence: K, V [len, heads, dim] in 64 bits, as stored
        shape = (pages, heads, page, dim)
        k, v = (np.full(shape, stale, np.float16 if fmt == "f16" else np.float64) for _ in range(2))
        if fmt == "q8":
            k, v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
            ks, vs = (np.full(shape[:3], stale, np.float32) for _ in range(2))
        for b, n in enumerate(lens):
            kv = []
            for data, scale in ((k, ks), (v, vs)) if fmt == "q8" else ((k, None), (v, None)):
                x = rng.standard_normal((n, heads, dim)).astype(np.float32) * np.exp(0.5 * rng.standard_normal((n, heads, 1)))
                if fmt == "q8":
                    code, d = q8_plain(x)
                    for p in range(n):
                        data[self.tables[b][p // page], :, p % page] = code[p]
                        scale[self.tables[b][p // page], :, p % page] = d[p]
                    kv.append(code.astype(np.float64) * d.astype(np.float64)[..., None])
                else:
                    x = x.astype(np.float16)
                    for p in range(n):
                        data[self.tables[b][p // page], :, p % page] = x[p]
                    kv.append(x.astype(np.float64))
            self.values.append(kv)
        self.cache.k.copy_(torch.from_numpy(k))
        self.cache.v.copy_(torch.from_numpy(v))
        if fmt == "q8":
            self.cache.k_scale.copy_(torch.from_numpy(ks))
            self.cache.v_scale.copy_(torch.from_numpy(vs))
        self.seqs = ops.Seqs.of(self.tables, new, lens)


def attend_plain(q, values, new, lens, scale, causal, unit_q, unit_w, unit_out):
    """(out, tolerance) in 64 bits; q: numpy [tokens, q heads, dim] as given to the operator."""
    q = q.astype(np.float64)
    tokens, qh, dim = q.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    t = 0
    for b, n in enumerate(new):
        k, v = values[b]
        length = lens[b]
        for i in range(n):
            see = min(length, max(0, length - n + i + 1)) if causal else length
            if see == 0:
                t += 1
                continue
            group = qh // k.shape[1]
            kk, vv = np.repeat(k[:see], group, 1), np.repeat(v[:see], group, 1)
            s = scale * np.einsum("hd,lhd->hl", q[t], kk)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o = np.einsum("hl,lhd->hd", p, vv)
            a = np.einsum("hl,lhd->hd", p, np.abs(vv))
            largest = np.abs(q[t]).max(-1)
            ds = abs(scale) * (unit_q * largest[:, None] * np.abs(kk).sum(-1).T
                               + dim * 2.0 ** -23 * np.einsum("hd,lhd->hl", np.abs(q[t]), np.abs(kk)))
            ds = ds.max(-1) + 2.0 ** -22 * (1 + np.abs(s).max(-1))  # and the exponential's argument
            out[t] = o
            tol[t] = unit_out * np.abs(o) + (2 * unit_w + 2 * ds[:, None] + see * 2.0 ** -23) * a
            tol[t] += see * 2.0 ** -31 * np.abs(vv).max() + (2.0 ** -25 if unit_out == 2.0 ** -11 else 0.0)
            t += 1
    return out, tol


UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def check_attend(ops, c, dtype, group=1, causal=True, scale=None, seqs=None, values=None, seed=1, q=None, out=None,
                 skip=None):
    torch = _torch()
    rng = np.random.default_rng(seed)
    if q is None:
        x = 2 * rng.standard_normal((sum(c.new), c.heads * group, c.dim))
        q = torch.from_numpy(x).to(dtype).cuda()
    got = c.cache.attend(seqs or c.seqs, q, scale=scale, causal=causal, out=out)
    single = dtype == torch.float32
    want, tol = attend_plain(q.cpu().double().numpy(), values or c.values, c.new, c.lens,
                             c.dim ** -0.5 if scale is None else scale, causal,
                             2.0 ** -21 if single else 2.0 ** -15, 2.0 ** -21 if single else 2.0 ** -11,
                             UNIT[str(got.dtype).split(".")[1]])
    got = got.cpu().double().numpy()
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol + 1e-30)
    if skip is not None:
        bad &= ~skip
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(got - want) / (tol + 1e-30)):.2f} of the tolerance"
    return got


# ---------------------------------------------------------------------------
# Write and read

@gpu_only
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_write_then_read(ops, dim, dtype):
    """Codes, scales and f16 numbers are exactly the format's; places of no new token keep what they held."""
    torch = _torch()
    dt = getattr(torch, dtype)
    for fmt in ("f16", "q8"):
        for heads, page, new, lens in ((1, 16, [1], [1]), (3, 16, [5, 0, 17, 1], [5, 9, 33, 64]), (16, 64, [130, 1, 63], [131, 300, 63])):
            c = Case(ops, fmt, heads, dim, page, new, lens, seed=dim + heads)
            tokens = sum(new)
            gen = torch.Generator().manual_seed(7)
            both = (torch.randn(tokens, 2, heads, dim, generator=gen) * torch.exp(2 * torch.randn(tokens, 2, heads, 1, generator=gen))).to(dt).cuda()
            both[0, 0, 0, :] = 0  # a row of zeros
            both[0, 1, 0, : dim // 2] = both[0, 1, 0, dim // 2:].abs().amax() / 2  # ratios of exactly 63.5
            before = [x.clone() if x is not None else None for x in (c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale)]
            c.cache.write(c.seqs, both[:, 0], both[:, 1])
            place = []
            for b, n in enumerate(new):
                place += [(c.tables[b][p // page], p % page) for p in range(lens[b] - n, lens[b])]
            for side, data, scale, old, old_scale in ((0, c.cache.k, c.cache.k_scale, before[0], before[2]), (1, c.cache.v, c.cache.v_scale, before[1], before[3])):
                x = both[:, side].float().cpu().numpy()
                want, want_scale = old.cpu().numpy(), None if old_scale is None else old_scale.cpu().numpy()
                code, d = q8_plain(x)
                for t, (pg, at) in enumerate(place):
                    want[pg, :, at] = code[t] if fmt == "q8" else x[t].astype(np.float16)
                    if fmt == "q8":
                        want_scale[pg, :, at] = d[t]
                np.testing.assert_array_equal(data.cpu().numpy(), want)
                if fmt == "q8":
                    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
            out = c.cache.read(c.seqs, dt)
            for side in (0, 1):
                x = both[:, side].float().cpu().numpy()
                code, d = q8_plain(x)
                value = code.astype(np.float32) * d[..., None] if fmt == "q8" else x.astype(np.float16).astype(np.float32)
                assert torch.equal(out[side].cpu(), torch.from_numpy(value).to(dt))


@gpu_only
def test_write_takes_any_strides_and_mixed_types(ops):
    torch = _torch()
    for fmt in ("f16", "q8"):
        c = Case(ops, fmt, 4, 64, 16, [9, 3], [20, 3])
        base = torch.randn(13, 4 * 64 * 3 + 5, device="cuda")
        k = base[:12, 3: 3 + 4 * 64].view(12, 4, 64)                        # rows that start at odd places
        v = torch.randn(4, 12, 64, device="cuda").half().transpose(0, 1)    # heads apart, another type
        c.cache.write(c.seqs, k, v)
        ok, ov = torch.full((12, 4, 64 + 1), 7.0, device="cuda")[..., :64], torch.empty(4, 12, 64, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
        c.cache.read(c.seqs, out=(ok, ov))
        for got, x in ((ok, k), (ov, v)):
            x = x.float().cpu().numpy()
            code, d = q8_plain(x)
            value = code.astype(np.float32) * d[..., None] if fmt == "q8" else x.astype(np.float16).astype(np.float32)
            assert torch.equal(got.cpu(), torch.from_numpy(value).to(got.dtype))


@gpu_only
def test_write_of_extreme_rows(ops):
    """Rows at the ends of f32's range, with infinities and with NaN, against the format's steps."""
    torch = _torch()
    x = torch.randn(8, 2, 32)
    x[0] *= 1e38
    x[1] *= 1e-42
    x[2] *= 1e-37
    x[3, 0, 5] = math.inf
    x[4, 1, 0] = math.nan
    x[5] = 0
    x[6, :, 1:] *= 1e-30  # one number far above the rest
    c = Case(ops, "q8", 2, 32, 16, [8], [8])
    c.cache.write(c.seqs, x.cuda(), x.cuda())
    code, d = q8_plain(x.numpy())
    got, scale = c.cache.k[c.tables[0][0], :, :8].cpu().numpy(), c.cache.k_scale[c.tables[0][0], :, :8].cpu().numpy()
    np.testing.assert_array_equal(scale.transpose(1, 0), d)
    np.testing.assert_array_equal(got.transpose(1, 0, 2), code)
    back = c.cache.read(c.seqs, torch.float32)[0].cpu()
    assert torch.isnan(back[3, 0]).all() and torch.isnan(back[4, 1]).all()
    assert torch.isfinite(back[3, 1]).all() and torch.isfinite(back[4, 0]).all()
    c = Case(ops, "f16", 2, 32, 16, [8], [8])
    c.cache.write(c.seqs, x.cuda(), x.cuda())
    assert torch.equal(c.cache.read(c.seqs, torch.float16)[0].cpu().view(torch.int16)[x.half().isfinite()],
                       x.half().view(torch.int16)[x.half().isfinite()])


@gpu_only
def test_places_that_do_not_exist(ops):
    """Tokens without a place are dropped by write, read as zeros, and are no keys: page numbers outside the cache,
    positions before the sequence's start or past its table, rows outside the call's."""
    torch = _torch()
    for fmt in ("f16", "q8"):
        c = Case(ops, fmt, 2, 16, 16, [20, 4, 2], [40, 3, 64], spare=0)
        table = c.seqs.tensors[0].clone()
        table[0, 1] = c.cache.pages + 5   # positions 16 .. 31 of sequence 0
        table[2, 0] = -3
        seqs = ops.Seqs(table, torch.tensor([0, 20, 24, 26], dtype=torch.int32, device="cuda"),
                        torch.tensor([40, 3, 65], dtype=torch.int32, device="cuda"), 20, 65, 26)  # 65: past the table
        before = c.cache.k.clone()
        x = torch.randn(26, 2, 16, device="cuda")
        c.cache.write(seqs, x, x)
        k, _ = c.cache.read(seqs, torch.float32)
        real = c.cache.k.float() if fmt == "f16" else c.cache.k.float() * c.cache.k_scale[..., None]
        for t in range(26):
            b = 0 if t < 20 else 1 if t < 24 else 2
            pos = (20 + t) if b == 0 else t - 21 if b == 1 else 63 + t - 24
            page = int(table[b, pos // 16]) if 0 <= pos < 16 * table.shape[1] else -1
            if 0 <= page < c.cache.pages:
                assert torch.equal(k[t], real[page, :, pos % 16])
            else:
                assert (k[t] == 0).all()
        touched = {int(table[b, p // 16]) for b, p in [(0, q) for q in range(32, 40)] + [(1, 0), (1, 1), (1, 2), (2, 63)]}
        for page in range(c.cache.pages):
            if page not in touched:
                assert torch.equal(c.cache.k[page].view(torch.int8), before[page].view(torch.int8))


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
def test_no_sequences(ops, fmt):
    """A call without sequences writes nothing and reads zeros, whether or not there are rows."""
    torch = _torch()
    cache = ops.PagedKV.empty(3, 2, 16, 32, fmt)
    cache.k.fill_(5)
    i32 = dict(dtype=torch.int32, device="cuda")
    for seqs in (ops.Seqs.of([], [], []), ops.Seqs(torch.zeros(0, 4, **i32), torch.zeros(1, **i32), torch.zeros(0, **i32))):
        out = tuple(torch.full((7, 2, 32), 3.0, device="cuda") for _ in range(2))
        cache.read(seqs, out=out)
        assert (out[0] == 0).all() and (out[1] == 0).all()
        cache.write(seqs, *(torch.ones(7, 2, 32, device="cuda") for _ in range(2)))
        assert (cache.k == 5).all() and (cache.v == 0).all()
        assert cache.read(ops.Seqs(*seqs.tensors, tokens=0))[0].shape == (0, 2, 32)
    # sequences without any room: positions that do not exist
    seqs = ops.Seqs(torch.zeros(2, 0, **i32), torch.tensor([0, 3, 4], **i32), torch.tensor([5, 1], **i32), tokens=4)
    cache.write(seqs, *(torch.ones(4, 2, 32, device="cuda") for _ in range(2)))
    assert (cache.k == 5).all() and all((x == 0).all() for x in cache.read(seqs))
    assert (cache.attend(seqs, torch.randn(4, 4, 32, device="cuda")) == 0).all()


# ---------------------------------------------------------------------------
# Attention

RAGGED = ([1, 0, 2, 7, 1, 3, 5, 1], [1, 5, 2, 40, 33, 130, 17, 300])


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_attend_few_rows(ops, fmt, dim, dtype, group):
    dt = getattr(_torch(), dtype)
    c = Case(ops, fmt, 2, dim, 16, *RAGGED, seed=dim + group)
    check_attend(ops, c, dt, group)
    if group == 3:
        check_attend(ops, c, dt, group, causal=False)


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("new,lens,heads,group,page", [
    ([65], [65], 1, 1, 16),                          # a bit over the kernel for few rows
    ([257], [257], 2, 1, 128),                       # two row tiles, the second with one row
    ([128, 1, 300, 0, 66], [700, 129, 300, 8, 127 + 66], 1, 1, 32),  # both kernels in one call
    ([40, 90], [400, 91], 2, 7, 64),
    ([300], [2100], 1, 1, 16),                       # keys cut over a cluster
])
def test_attend_many_rows(ops, fmt, dim, new, lens, heads, group, page):
    torch = _torch()
    c = Case(ops, fmt, heads, dim, page, new, lens, seed=sum(new))
    check_attend(ops, c, torch.float16, group)
    if dim == 64:
        check_attend(ops, c, torch.bfloat16, group, causal=False)
        check_attend(ops, c, torch.float32, group)


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
def test_attend_long_context(ops, fmt):
    """The split over 16 CTAs of a cluster, and many row tiles that all run."""
    torch = _torch()
    c = Case(ops, fmt, 1, 64, 256, [1, 2], [9001, 4095])
    check_attend(ops, c, torch.float16, 4)
    check_attend(ops, c, torch.float32, 4)


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("new", [6, 200])
def test_rows_that_see_nothing(ops, fmt, new):
    """Fewer positions than new tokens, and no positions at all: zeros."""
    torch = _torch()
    c = Case(ops, fmt, 2, 64, 16, [new, 3, new], [new - 4, 0, new])
    for dt in (torch.float16, torch.float32):
        got = check_attend(ops, c, dt, 2)
        assert (got[: 4] == 0).all() and (got[new: new + 3] == 0).all()


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("new", [9, 150])
def test_masked_values_never_reach_a_row(ops, fmt, new):
    """NaN and infinities in the K and V of later tokens leave earlier tokens' rows alone; rows that see them are not
    finite where V is not."""
    torch = _torch()
    n, length = new, new + 37
    c = Case(ops, fmt, 1, 64, 16, [n], [length])
    bad = length - 5  # seen by the last five tokens alone
    page, at = c.tables[0][bad // 16], bad % 16
    page2, at2 = c.tables[0][(bad + 2) // 16], (bad + 2) % 16
    if fmt == "f16":
        c.cache.v[page, 0, at, 3] = math.nan
        c.cache.v[page2, 0, at2, 7] = math.inf
        c.cache.k[page2, 0, at2, 0] = math.nan
    else:
        c.cache.v_scale[page, 0, at] = math.nan
        c.cache.k_scale[page2, 0, at2] = math.nan
    q = torch.randn(n, 1, 64, device="cuda").half()
    clean = [[x.copy() for x in kv] for kv in c.values]
    keep = np.zeros((n, 1, 64), bool)
    keep[n - 5:] = True
    got = check_attend(ops, c, torch.float16, values=clean, q=q, skip=keep)
    assert np.isfinite(got[: n - 5]).all()
    assert not np.isfinite(got[n - 5:, 0, 3]).any()
    if fmt == "f16":
        assert np.isfinite(got[n - 5: n - 3, 0, :3]).all()
    check = c.cache.attend(c.seqs, q.float())[: n - 5]
    assert torch.isfinite(check).all()


@gpu_only
@pytest.mark.parametrize("new,first", [(9, 5), (60, 20), (150, 30), (512, 400), (700, 130)])
@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("size", [math.nan, math.inf, 2.0 ** 8, 2.0 ** 12, 2.0 ** 16, 2.0 ** 40, 1e36])
def test_scales_of_later_tokens_never_reach_a_row(ops, new, first, dim, size):
    """However large V's scales are from new token `first` on, and where they are no numbers: the tokens before see none
    of them, and later ones what the definition says of finite scales."""
    torch = _torch()
    length = new + 37
    c = Case(ops, "q8", 1, dim, 16, [new], [length], seed=new)
    for p in range(length - new + first, length):
        page, at = c.tables[0][p // 16], p % 16
        c.cache.v_scale[page, 0, at] *= size
        with np.errstate(invalid="ignore"):
            c.values[0][1][p] = c.cache.v[page, :, at].cpu().double().numpy() * c.cache.v_scale[page, :, at].cpu().double().numpy()[:, None]
    later = np.zeros((new, 2, dim), bool)
    later[first:] = not math.isfinite(size)
    c.values = [[np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) for x in kv] for kv in c.values]
    for dt in (torch.float16, torch.bfloat16, torch.float32):
        q = torch.randn(new, 2, dim, device="cuda").to(dt)
        out = torch.empty(new, 2, dim, device="cuda")
        got = check_attend(ops, c, dt, 2, q=q, out=out, skip=later)
        assert np.isfinite(got[:first]).all()
        if not math.isfinite(size):  # a code of 0 times an infinity is no number either
            assert not np.isfinite(got[first:]).any()


@gpu_only
def test_a_score_below_all_numbers_beside_a_hole(ops):
    """Two rows of a tile, of which one's score of a key is -inf, where V's scale is large and the page behind is missing:
    the other row's later keys keep their weight."""
    torch = _torch()
    c = Case(ops, "q8", 1, 32, 16, [1], [700], stale=0.0)
    page, at = c.tables[0][0], 3
    c.cache.k[page, 0, at] = 100
    c.cache.k_scale[page, 0, at] = 1e25
    c.cache.v_scale[page, 0, at] *= 2.0 ** 40
    table = c.seqs.tensors[0].clone()
    table[0, 1] = c.cache.pages
    seqs = ops.Seqs(table, *c.seqs.tensors[1:], 1, 700)
    q = torch.empty(1, 2, 32, device="cuda")
    q[0, 0], q[0, 1] = -1e20, -5e-28
    c.values[0][0][at, 0] = 100 * float(c.cache.k_scale[page, 0, at])
    c.values[0][1][at, 0] *= 2.0 ** 40
    short = [[np.delete(x, range(16, 32), 0) for x in c.values[0]]]
    for dt in (torch.float32, torch.bfloat16):
        units = (2.0 ** -21, 2.0 ** -21, 2.0 ** -24) if dt == torch.float32 else (2.0 ** -15, 2.0 ** -11, 2.0 ** -24)
        want, tol = attend_plain(q.to(dt).cpu().double().numpy(), short, [1], [684], 32 ** -0.5, True, *units)
        got = c.cache.attend(seqs, q.to(dt), out=torch.empty_like(q)).cpu().double().numpy()
        assert (np.abs(got - want) <= tol)[0, 1].all(), (np.abs(got - want) / tol)[0, 1].max()


@gpu_only
@pytest.mark.parametrize("new,length", [(1, 40), (3, 9001), (20, 700), (150, 160), (300, 2100)])
@pytest.mark.parametrize("size", [1e36, 1e-34])
def test_values_near_the_ends_of_the_range(ops, new, length, size):
    """Values of 1e37 and of 1e-34: the outputs are as large, the sums before the division by the weights' would not be."""
    torch = _torch()
    c = Case(ops, "q8", 2, 64, 64, [new], [length])
    c.cache.v_scale *= size
    v = [c.cache.v[c.tables[0][p // 64], :, p % 64].cpu().double().numpy()
         * c.cache.v_scale[c.tables[0][p // 64], :, p % 64].cpu().double().numpy()[:, None] for p in range(length)]
    c.values[0][1] = np.stack(v)
    for dt in (torch.float16, torch.float32):
        q = torch.randn(new, 4, 64, device="cuda").to(dt)
        check_attend(ops, c, dt, 2, q=q, out=torch.empty(new, 4, 64, device="cuda"))


@gpu_only
@pytest.mark.parametrize("new,first", [(512, 400), (1000, 390)])
def test_scales_without_a_number_for_long(ops, new, first):
    """Whole tiles of later tokens whose V scales are NaN: the tokens before keep their values."""
    torch = _torch()
    c = Case(ops, "q8", 1, 64, 128, [new], [new])
    clean = [[x.copy() for x in kv] for kv in c.values]
    for p in range(first, new):
        c.cache.v_scale[c.tables[0][p // 128], 0, p % 128] = math.nan
    later = np.zeros((new, 1, 64), bool)
    later[first:] = True
    q = torch.randn(new, 1, 64, device="cuda").half()
    got = check_attend(ops, c, torch.float16, q=q, values=clean, skip=later)
    assert np.isnan(got[first:]).all()


@gpu_only
@pytest.mark.parametrize("new", [9, 150, 300, 700])
@pytest.mark.parametrize("dim", [16, 128])
def test_infinite_values_keep_their_sign(ops, new, dim):
    """A row that sees an infinite V gets that infinity in its dim, one that sees both signs NaN, the others neither."""
    torch = _torch()
    length = new + 37
    c = Case(ops, "f16", 1, dim, 16, [new], [length])
    for at, d, x in ((3, 9, math.inf), (length - 7, 2, math.inf), (length - 4, 2, -math.inf), (length - 4, 5, -math.inf)):
        c.cache.v[c.tables[0][at // 16], 0, at % 16, d] = x
        c.values[0][1][at, 0, d] = x
    q = 0.1 * torch.randn(new, 1, dim, device="cuda").half()
    with np.errstate(invalid="ignore"):
        want, _ = attend_plain(q.cpu().double().numpy(), c.values, c.new, c.lens, dim ** -0.5, True, 2.0 ** -15, 2.0 ** -11, 2.0 ** -11)
    got = c.cache.attend(c.seqs, q).cpu().double().numpy()
    fin = np.isfinite(want)
    assert np.isposinf(want[:, 0, 9]).all() and np.isneginf(want[-1, 0, 5]) and np.isnan(want[-1, 0, 2]) and np.isposinf(want[-6, 0, 2])
    np.testing.assert_array_equal(got[~fin], want[~fin])
    assert np.isfinite(got[fin]).all()
    _, tol = attend_plain(q.cpu().double().numpy(), [[np.nan_to_num(x, posinf=0.0, neginf=0.0) for x in kv] for kv in c.values], c.new,
                          c.lens, dim ** -0.5, True, 2.0 ** -15, 2.0 ** -11, 2.0 ** -11)
    assert (np.abs(got[fin] - want[fin]) <= tol[fin]).all()


@gpu_only
@pytest.mark.parametrize("new", [1, 9, 150, 300])
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_infinite_values_keep_their_sign_for_wider_queries(ops, new, dim, dtype):
    """As above where the weights have two parts, or q is scaled: infinities that all rows see, and that some do."""
    torch = _torch()
    dt, length = getattr(torch, dtype), new + 70
    c = Case(ops, "f16", 1, dim, 16, [new], [length])
    for at, d, x in ((3, 9, math.inf), (40, 11, -math.inf), (41, 12, math.inf), (50, 12, -math.inf), (length - 1, 5, -math.inf),
                     (60, 13, math.nan)):
        c.cache.v[c.tables[0][at // 16], 0, at % 16, d] = x
        c.values[0][1][at, 0, d] = x
    q = (0.1 * torch.randn(new, 2, dim, device="cuda")).to(dt)
    single = dt == torch.float32
    units = (2.0 ** -21, 2.0 ** -21, 2.0 ** -24) if single else (2.0 ** -15, 2.0 ** -11, 2.0 ** -24)
    with np.errstate(invalid="ignore"):
        want, _ = attend_plain(q.cpu().double().numpy(), c.values, c.new, c.lens, dim ** -0.5, True, *units)
    got = c.cache.attend(c.seqs, q, out=torch.empty(new, 2, dim, device="cuda")).cpu().double().numpy()
    fin = np.isfinite(want)
    assert np.isposinf(want[..., 9]).all() and np.isneginf(want[..., 11]).all() and np.isnan(want[..., 12]).all() and np.isneginf(want[-1, :, 5]).all()
    np.testing.assert_array_equal(got[~fin], want[~fin])
    _, tol = attend_plain(q.cpu().double().numpy(), [[np.nan_to_num(x, posinf=0.0, neginf=0.0) for x in kv] for kv in c.values], c.new,
                          c.lens, dim ** -0.5, True, *units)
    assert (np.abs(got[fin] - want[fin]) <= tol[fin]).all()


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("new", [3, 100])
def test_attend_holes_hints_and_scales(ops, fmt, new):
    torch = _torch()
    c = Case(ops, fmt, 2, 32, 16, [new, 1], [new + 100, 70])
    # a page outside the cache takes its positions out of the sequence
    table = c.seqs.tensors[0].clone()
    table[0, 2] = c.cache.pages
    seqs = ops.Seqs(table, *c.seqs.tensors[1:], new, new + 100)
    torch_q = torch.randn(new + 1, 4, 32, device="cuda").half()
    got = c.cache.attend(seqs, torch_q).cpu().double().numpy()
    # the same with those keys cut out, causally (they all lie before the new tokens)
    short = [np.delete(x, range(32, 48), 0) for x in c.values[0]]
    want, tol = attend_plain(torch_q.cpu().double().numpy(), [short, c.values[1]], c.new, [new + 84, 70], 32 ** -0.5, True,
                             2.0 ** -15, 2.0 ** -11, 2.0 ** -11)
    assert (np.abs(got - want) <= tol).all()
    # bounds that are too small, and none
    for bounds in ((1, 1), (None, None)):
        check_attend(ops, c, torch.float16, 2, seqs=ops.Seqs(*c.seqs.tensors, *bounds))
        check_attend(ops, c, torch.float32, 2, seqs=ops.Seqs(*c.seqs.tensors, *bounds))
    for scale in (0.0, -0.3, 4.0):
        check_attend(ops, c, torch.float16, 2, scale=scale)


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("new,lens,rows,bound", [
    ([300, 1], [400, 90], 1024, 300),     # rows to spare behind the sequences'
    ([300, 1], [400, 90], 602, 301),
    ([40], [140], 512, 512),
    ([1], [77], 512, 512),
    ([2, 0, 64, 65], [5, 0, 90, 70], 2048, 512),
    ([599, 1], [640, 50], 600, 300),      # a bound that is too small
    ([700, 1, 7], [800, 500, 7], 708, 200),
])
def test_every_sequence_is_computed(ops, fmt, new, lens, rows, bound):
    """Whatever the bound and the number of rows say of the sequences' lengths: no row of theirs keeps what out held."""
    torch = _torch()
    c = Case(ops, fmt, 2, 64, 16, new, lens, seed=rows)
    seqs = ops.Seqs(*c.seqs.tensors, bound, max(lens))
    spare = np.zeros((rows, 4, 64), bool)
    spare[sum(new):] = True
    for dt in (torch.float16, torch.bfloat16, torch.float32):
        q = torch.randn(rows, 4, 64, device="cuda").to(dt)
        check_attend(ops, c, dt, 2, seqs=seqs, q=q, out=torch.full_like(q, math.nan), skip=spare)


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("new,rows", [([3, 4], 5), ([20, 30], 35), ([300, 300], 450), ([300, 5], 302)])
def test_more_new_tokens_than_rows(ops, fmt, new, rows):
    """A token whose row is not one of the call's still has its position: the others see what they saw with it, as in
    the write and the read."""
    torch = _torch()
    c = Case(ops, fmt, 2, 32, 16, new, [n + 9 for n in new])
    for dt in (torch.float16, torch.float32):
        q = torch.randn(sum(new), 4, 32, device="cuda").to(dt)
        want, tol = attend_plain(q.cpu().double().numpy(), c.values, c.new, c.lens, 32 ** -0.5, True,
                                 *((2.0 ** -21,) * 2 if dt == torch.float32 else (2.0 ** -15, 2.0 ** -11)), UNIT[str(dt).split(".")[1]])
        got = c.cache.attend(c.seqs, q[:rows]).cpu().double().numpy()
        assert (np.abs(got - want[:rows]) <= tol[:rows] + 1e-30).all()
    for got, want in zip(c.cache.read(c.seqs, out=tuple(torch.empty(rows, 2, 32, device="cuda") for _ in range(2))),
                         c.cache.read(c.seqs, torch.float32)):
        assert torch.equal(got, want[:rows])


@gpu_only
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("new,before,after,bound", [
    ([1, 3], 0, 5, 3), ([1, 3], 2, 0, 3), ([300], 7, 213, 300), ([300, 40, 1], 1, 700, 300), ([300, 2], 0, 900, 300), ([0, 0], 0, 9, 0), ([], 0, 40, 0)])
def test_rows_of_no_sequence_are_zeros(ops, dtype, new, before, after, bound):
    """Rows before the first sequence's and behind the last one's, whichever kernel runs; places between rows stay."""
    torch = _torch()
    dt = getattr(torch, dtype)
    c = Case(ops, "q8", 2, 32, 16, new, [n + 50 for n in new])
    table, start, length = c.seqs.tensors
    seqs = ops.Seqs(table, start + before, length, bound, max([n + 50 for n in new], default=0))
    tokens = before + sum(new) + after
    q = torch.randn(tokens, 6, 32, device="cuda").to(dt)
    for wide in (32, 33):  # rows that allow wide stores, and that do not
        out = torch.full((tokens, 6, wide + 8), math.nan, device="cuda", dtype=dt)
        c.cache.attend(seqs, q, out=out[..., :32])
        got = out[..., :32].float()
        assert (got[:before] == 0).all() and (got[before + sum(new):] == 0).all() and torch.isnan(out[..., 32:]).all()
        mine = slice(before, before + sum(new))
        want, tol = attend_plain(q[mine].cpu().double().numpy(), c.values, c.new, c.lens, 32 ** -0.5, True,
                                 *((2.0 ** -21,) * 2 if dt == torch.float32 else (2.0 ** -15, 2.0 ** -11)), UNIT[dtype])
        assert (np.abs(got[mine].cpu().double().numpy() - want) <= tol + 1e-30).all()
    assert (c.cache.attend(seqs, q)[before + sum(new):] == 0).all()


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
def test_graph_replayed_over_other_lengths(ops, fmt):
    """A step captured for up to 512 new tokens, replayed for the last chunk of a prompt and for single tokens."""
    torch = _torch()
    c = Case(ops, fmt, 2, 64, 16, [512, 512], [700, 600])
    start, length = (x.clone() for x in c.seqs.tensors[1:])
    seqs = ops.Seqs(c.seqs.tensors[0], start, length, 512, 700)
    q = torch.randn(1024, 2, 64, device="cuda").half()
    out = torch.empty_like(q)
    c.cache.attend(seqs, q, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.cache.attend(seqs, q, out=out)
    for new, lens in (([512, 512], [700, 600]), ([40, 512], [700, 600]), ([512, 1], [600, 600]), ([40, 1], [40, 555]), ([1, 1], [1, 600])):
        start.copy_(torch.tensor([0, new[0], sum(new)], dtype=torch.int32))
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(math.nan)
        graph.replay()
        want, tol = attend_plain(q.cpu().double().numpy(), [[x[:n] for x in kv] for kv, n in zip(c.values, lens)], new, lens,
                                 64 ** -0.5, True, 2.0 ** -15, 2.0 ** -11, 2.0 ** -11)
        got = out.cpu().double().numpy()
        assert (np.abs(got - want) <= tol)[: sum(new)].all()


@gpu_only
@pytest.mark.parametrize("new", [2, 130])
def test_attend_strides_and_types(ops, new):
    torch = _torch()
    c = Case(ops, "q8", 2, 64, 32, [new], [new + 50])
    for shift in (1, 4, 8):  # rows at odd places, at four and at eight numbers
        for dt in (torch.float16, torch.bfloat16, torch.float32):
            wide = torch.randn(4, new, 64 * 3 + shift, device="cuda").to(dt)
            q = wide[..., shift: shift + 64].transpose(0, 1)
            for out_dt in (torch.float16, torch.float32):
                out = torch.full((new, 4, 64 + shift), 5.0, device="cuda", dtype=out_dt)
                check_attend(ops, c, dt, 2, q=q, out=out[..., :64])
                assert (out[..., 64:] == 5).all()


@gpu_only
@pytest.mark.parametrize("magnitude", [1e-30, 1e-6, 3e4, 1e30])
def test_attend_query_and_cache_ranges(ops, magnitude):
    """Queries and 8-bit scales far from 1: their product is what counts."""
    torch = _torch()
    for new in (3, 80):
        c = Case(ops, "q8", 1, 32, 16, [new], [new + 20])
        c.cache.k_scale /= magnitude
        k = []
        for p in range(c.lens[0]):
            page, at = c.tables[0][p // 16], p % 16
            k.append(c.cache.k[page, :, at].cpu().double().numpy() * c.cache.k_scale[page, :, at].cpu().double().numpy()[:, None])
        c.values[0][0] = np.stack(k)
        q = torch.randn(new, 1, 32, device="cuda") * magnitude
        check_attend(ops, c, torch.float32, q=q)
        if magnitude != 3e4:
            check_attend(ops, c, torch.bfloat16, q=q.bfloat16())
        c = Case(ops, "q8", 1, 32, 16, [new], [new + 20])
        for p in range(c.lens[0]):  # V's scales over a wide range
            c.cache.v_scale[c.tables[0][p // 16], :, p % 16] *= magnitude if p % 3 else 1.0
        v = [c.cache.v[c.tables[0][p // 16], :, p % 16].cpu().double().numpy()
             * c.cache.v_scale[c.tables[0][p // 16], :, p % 16].cpu().double().numpy()[:, None] for p in range(c.lens[0])]
        c.values[0][1] = np.stack(v)
        check_attend(ops, c, torch.float32)
        check_attend(ops, c, torch.bfloat16)


@gpu_only
@pytest.mark.parametrize("new", [3, 80])
@pytest.mark.parametrize("magnitude", [1e-31, 4e-31])
def test_tiny_queries_count(ops, new, magnitude):
    """Queries below 1e-30 over keys as large as they are small."""
    torch = _torch()
    c = Case(ops, "q8", 1, 32, 16, [new], [new + 20])
    c.cache.k_scale /= magnitude
    c.values[0][0] = np.stack([c.cache.k[c.tables[0][p // 16], :, p % 16].cpu().double().numpy()
                               * c.cache.k_scale[c.tables[0][p // 16], :, p % 16].cpu().double().numpy()[:, None] for p in range(new + 20)])
    q = torch.randn(new, 1, 32, device="cuda") * magnitude
    check_attend(ops, c, torch.float32, q=q)
    check_attend(ops, c, torch.bfloat16, q=q.bfloat16())


@gpu_only
@pytest.mark.parametrize("new", [3, 300])
@pytest.mark.parametrize("scale", [0.0, -0.0])
def test_a_scale_of_zero(ops, new, scale):
    """Every key that is seen counts alike, however large the products are."""
    torch = _torch()
    for fmt, size in (("q8", 1e12), ("f16", 1.0)):
        c = Case(ops, fmt, 1, 32, 16, [new], [new + 20])
        if fmt == "q8":
            c.cache.k_scale *= size
        for dt, top in ((torch.float32, 1e22), (torch.bfloat16, 1e22), (torch.float16, 1e4)):
            q = (torch.randn(new, 1, 32, device="cuda") * (top if fmt == "q8" else 1.0)).to(dt)
            check_attend(ops, c, dt, q=q, scale=scale)


@gpu_only
def test_cache_beyond_32_bit_offsets(ops):
    """Places whose numbers lie past 2^31 of a side."""
    torch = _torch()
    pages = (1 << 31) // (16 * 64 * 128) + 300
    cache = ops.PagedKV(*(torch.zeros(pages, 16, 64, 128, dtype=torch.int8, device="cuda") for _ in range(2)),
                        *(torch.zeros(pages, 16, 64, device="cuda") for _ in range(2)))
    small = Case(ops, "q8", 16, 128, 64, [70, 1], [200, 130])
    tables = [[pages - 1 - p for p in t] for t in small.tables]
    for mine, theirs in zip(small.tables, tables):
        for a, b in zip(mine, theirs):
            for name in ("k", "v", "k_scale", "v_scale"):
                getattr(cache, name)[b] = getattr(small.cache, name)[a]
    seqs = ops.Seqs.of(tables, small.new, small.lens)
    q = torch.randn(71, 16, 128, device="cuda").half()
    assert torch.equal(cache.attend(seqs, q), small.cache.attend(small.seqs, q))
    x = torch.randn(71, 16, 128, device="cuda")
    cache.write(seqs, x, x)
    small.cache.write(small.seqs, x, x)
    for a, b in zip(cache.read(seqs, torch.float32), small.cache.read(small.seqs, torch.float32)):
        assert torch.equal(a, b)


@gpu_only
def test_streams_graphs_and_repeats(ops):
    """On another stream and inside a captured graph the same bits come out, time after time."""
    torch = _torch()
    c = Case(ops, "q8", 4, 64, 16, [3, 100, 1], [500, 700, 9])
    q = torch.randn(104, 8, 64, device="cuda").half()
    x = torch.randn(104, 4, 64, device="cuda")
    logits = torch.randn(5, 5003, device="cuda")
    rules = ops.LogitRules(history=torch.randint(0, 5003, (5, 300), dtype=torch.int32, device="cuda"),
                           repetition=torch.full((5,), 1.3, device="cuda"))

    def step():
        c.cache.write(c.seqs, x, x)
        return (c.cache.attend(c.seqs, q), *c.cache.read(c.seqs, torch.float32), *rules.choose(logits))

    want = [y.clone() for y in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            for a, b in zip(step(), want):
                assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for y in got:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


GAVE_UP = """
import sys
import torch
from malaga_b200 import _lib, ops

fmt, parts = sys.argv[1], int(sys.argv[2])
new, length = (300, 2100) if parts > 1 else (1100, 1100)
pages = -(-length // 16)
cache = ops.PagedKV.empty(2 * pages, 4 if parts > 1 else 16, 16, 64, fmt)
seqs = ops.Seqs.of([list(range(pages)), list(range(pages, 2 * pages))], [new, new], [length, length])
q = torch.randn(2 * new, cache.heads, 64, device="cuda").half()
out = cache.attend(seqs, q)
try:
    cache.check()
    raise SystemExit("no error")
except _lib.MgbError as e:
    assert e.code == _lib.MGB_ERR_CUDA and "ran out of time" in str(e), e
cache.check()  # told once
lost = out.isnan().flatten(1).any(1)
# the first CTA has rows of the first sequence's first head alone; the caches hold zeros, and so do the other rows
assert lost[:new].any() and not lost[new:].any() and not out[:, 1:].isnan().any() and (out[:, 1:] == 0).all()
assert (torch.arange(1000, device="cuda").sum() == 499500).item()
"""


@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("parts,stage", [(1, 0), (1, 1), (8, 1)])
def test_a_wait_that_runs_out_is_told(ops, fmt, parts, stage):
    """One CTA waits for an arrival of keys that never comes and gives up: the kernel ends, its rows are NaN,
    mgb_kv_status says so once, and the device goes on. In a process of its own, since the hook is read once."""
    import os
    import subprocess
    import sys

    env = dict(os.environ, MGB_TEST_WITHHOLD_KEYS=str(stage))
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", GAVE_UP, fmt, str(parts)], env=env, cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@gpu_only
def test_status_is_good(ops):
    c = Case(ops, "q8", 2, 64, 16, [300, 1], [400, 50])
    c.cache.attend(c.seqs, _torch().randn(301, 2, 64, device="cuda").half())
    c.cache.check()


@gpu_only
def test_mixed_calls_read_what_was_just_written(ops):
    """Both kernels of a call of unlike sequences start from what the kernel right before it wrote (queries, lengths,
    page tables, the cache), on two streams at once and in a replayed graph."""
    torch = _torch()
    c = Case(ops, "f16", 4, 64, 16, [300, 1, 7, 20], [900, 700, 400, 333])
    steps = 24
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(steps, 328, 4, 64, device="cuda", generator=gen).half()
    k = torch.randn(steps, 328, 4, 64, device="cuda", generator=gen).half()
    less = torch.randint(0, 90, (steps, 4), device="cuda", generator=gen, dtype=torch.int32)

    class Side:
        def __init__(self):
            self.cache = ops.PagedKV(c.cache.k.clone(), c.cache.v.clone())
            self.table, self.start, self.length = (x.clone() for x in c.seqs.tensors)
            self.seqs = ops.Seqs(self.table, self.start, self.length, 300, 900)
            self.q, self.k, self.out = torch.zeros_like(q[0]), torch.zeros_like(k[0]), torch.zeros_like(q[0])

        def step(self, i, settle):
            """i: the step's number on the device, [1]."""
            pages = c.seqs.tensors[0].shape[1]
            self.cache.write(self.seqs, self.k, self.k)
            torch.index_select(k, 0, i, out=self.k[None])
            self.length.copy_((c.seqs.tensors[2][None] - less[i])[0])
            self.table[1, : pages // 2].copy_(c.seqs.tensors[0][1][: pages // 2].roll(3))
            torch.index_select(q, 0, i, out=self.q[None])
            if settle:
                torch.cuda.synchronize()
            self.cache.attend(self.seqs, self.q, out=self.out)
            return self.out

    numbers = torch.arange(steps, device="cuda")
    side, want = Side(), []
    for i in range(steps):
        want.append(side.step(numbers[i: i + 1], True).clone())
        torch.cuda.synchronize()
    streams, sides, got = [torch.cuda.Stream() for _ in range(2)], [Side(), Side()], [[], []]
    torch.cuda.synchronize()
    for i in range(steps):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[s].append(sides[s].step(numbers[i: i + 1], False).clone())
    torch.cuda.synchronize()
    for s in range(2):
        for a, b in zip(got[s], want):
            assert torch.equal(a, b)
    side, at = Side(), torch.zeros(1, dtype=torch.int64, device="cuda")
    fresh = [x.clone() for x in (side.cache.k, side.cache.v, side.k, side.length, side.table)]
    side.step(at, False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.step(at, False)
    for x, y in zip((side.cache.k, side.cache.v, side.k, side.length, side.table), fresh):
        x.copy_(y)
    for i in range(steps):
        at.fill_(i)
        graph.replay()
        assert torch.equal(side.out, want[i])


# ---------------------------------------------------------------------------
# Logits

def logits_plain(x, kw):
    """Adjusted logits in 64 bits and their tolerance before the type's rounding."""
    y = x.astype(np.float64)
    rows, vocab = y.shape
    tol = np.zeros(y.shape)
    for r in range(rows):
        if kw.get("history") is not None:
            h = kw["history"][r]
            if kw.get("history_len") is not None:
                h = h[: max(0, kw["history_len"][r])]
            ids, c = np.unique(h[(h >= 0) & (h < vocab)], return_counts=True)
            rep, freq, pres = (float(kw[n][r]) if kw.get(n) is not None else d for n, d in (("repetition", 1.0), ("frequency", 0.0), ("presence", 0.0)))
            z = y[r, ids]
            y[r, ids] = np.where(z > 0, z / rep, z * rep) - (freq * c + pres)
        if kw.get("bias") is not None:
            for i, v in zip(kw["bias_ids"][r], kw["bias"][r]):
                if 0 <= i < vocab:
                    y[r, i] += float(v)
                    tol[r, i] += 2.0 ** -23 * len(kw["bias"][r]) * abs(float(v))  # their own sum is in 32 bits
        if kw.get("allow") is not None:
            g = kw["allow_row"][r] if kw.get("allow_row") is not None else 0
            if 0 <= g < len(kw["allow"]):
                bits = np.unpackbits(np.ascontiguousarray(kw["allow"][g]).view(np.uint8), bitorder="little")[:vocab]
                y[r, bits == 0] = -np.inf
                tol[r, bits == 0] = 0
    return y, tol


def check_logits(ops, x, kw, dtype, in_place=False):
    """Choice and adjusted logits. A sum of exponentials has 2^-21 (the exponential) + 2^-23 |y - top| of relative error
    where it matters (within 32 of the top), and y is rounded to 2^-24 once."""
    torch = _torch()
    xt = x if isinstance(x, torch.Tensor) else torch.from_numpy(x).to(dtype).cuda()
    plain = xt.float().cpu().numpy()
    rules = ops.LogitRules(**{k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in kw.items() if v is not None})
    want, tol = logits_plain(plain, kw)
    first = rules.choose(xt)
    out = xt if in_place else torch.full_like(xt, 77.0)
    ids, logp, adjusted = rules.choose(xt, out)
    assert adjusted is out and torch.equal(ids, first[0]) and torch.equal(logp.view(torch.int32), first[1].view(torch.int32))
    got = adjusted.double().cpu().numpy()
    unit = UNIT[str(dtype).split(".")[1]]
    small = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -133}[str(dtype).split(".")[1]]
    fin = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - want)[fin] <= (unit * np.abs(want) + 2.0 ** -24 * np.abs(want) + tol + small)[fin]).all()
    ids, logp = ids.cpu().numpy(), logp.double().cpu().numpy()
    for r in range(len(want)):
        y = np.where(np.isnan(want[r]), -np.inf, want[r])
        top = y.max() if y.size else -np.inf
        if top == -np.inf:
            assert ids[r] == -1 and logp[r] == -np.inf
            continue
        near = 2.0 ** -22 * np.abs(top) + tol[r].max() if np.isfinite(top) else 0
        assert y[ids[r]] >= top - near
        if near == 0 or (y >= top - near).sum() == 1:
            assert ids[r] == int(np.argmax(y))
        if np.isfinite(top):
            ref = -np.log1p(np.exp(np.delete(y, np.argmax(y)) - top).sum())
            share = 1 - np.exp(ref)
            limit = share * (2.0 ** -21 + 32 * 2.0 ** -23 + 2.0 ** -22 * np.abs(y[np.isfinite(y) & (y > top - 32)]).max()) + 2.0 ** -23 * abs(ref) + 2 * share * tol[r].max()
            assert abs(logp[r] - ref) <= limit + 1e-15, (logp[r], ref, limit)
    return ids


def some_rules(rng, rows, vocab, history=40, bias=12, grammars=3):
    h = rng.integers(-2, vocab + 2, (rows, history)).astype(np.int32)
    h[:, history // 2:] = h[:, : history - history // 2]  # repeats
    bits = rng.random((grammars, (vocab + 31) // 32 * 32)) < 0.4
    allow = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    ids = rng.integers(-1, vocab + 1, (rows, bias)).astype(np.int32)
    ids[:, -3:] = ids[:, :1]  # three more entries of one token
    return dict(history=h, history_len=rng.integers(0, history + 1, rows).astype(np.int32),
                repetition=rng.uniform(0.7, 1.6, rows).astype(np.float32), frequency=rng.uniform(-0.2, 0.6, rows).astype(np.float32),
                presence=rng.uniform(0, 0.5, rows).astype(np.float32), bias_ids=ids,
                bias=rng.normal(0, 3, (rows, bias)).astype(np.float32), allow=allow,
                allow_row=rng.integers(-1, grammars + 1, rows).astype(np.int32))


@gpu_only
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 7), (3, 33), (5, 64), (40, 1000), (1, 4097), (3, 8193), (2, 70001), (310, 35001)])
def test_logits(ops, dtype, rows, vocab):
    dt = getattr(_torch(), dtype)
    rng = np.random.default_rng(vocab)
    x = 4 * rng.standard_normal((rows, vocab)).astype(np.float32)
    rules = some_rules(rng, rows, vocab)
    check_logits(ops, x, rules, dt)
    if rows < 300:
        check_logits(ops, x, {}, dt)
        check_logits(ops, x, {k: rules[k] for k in ("history", "repetition")}, dt, in_place=True)
        check_logits(ops, x, {k: rules[k] for k in ("bias_ids", "bias")}, dt)
        check_logits(ops, x, {"allow": rules["allow"]}, dt, in_place=True)


@gpu_only
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_logits_rows_at_odd_places(ops, dtype):
    torch = _torch()
    dt, rng = getattr(torch, dtype), np.random.default_rng(3)
    for shift, vocab in ((1, 5003), (3, 20001), (5, 11)):
        wide = torch.randn(4, vocab + 9, device="cuda").to(dt)
        x = wide[:, shift: shift + vocab]
        check_logits(ops, x, some_rules(rng, 4, vocab), dt)
        check_logits(ops, x, some_rules(rng, 4, vocab), dt, in_place=True)


@gpu_only
def test_logits_long_history(ops):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((3, 40000)).astype(np.float32)
    check_logits(ops, x, some_rules(rng, 3, 40000, history=20000, bias=700), _torch().float32)
    check_logits(ops, np.repeat(x, 60, 0), some_rules(rng, 180, 40000, history=3000), _torch().float32)


@gpu_only
def test_logits_ties_masks_and_non_finite(ops):
    torch = _torch()
    x = np.zeros((9, 3001), np.float32)
    x[0, [2900, 17, 400]] = 3.0                      # the lowest of equals
    x[1, :] = -np.inf                                # nothing to choose
    x[2, :] = np.nan
    x[3, 5] = np.nan
    x[3, 9] = 2.0
    x[4, 100] = np.inf
    x[5, [7, 2000]] = np.inf
    x[6, :] = -np.inf
    x[6, 3000] = -5.0                                # a choice that is certain
    x[7, 11] = np.finfo(np.float32).max              # masked below
    allow = np.zeros((2, 94), np.int32)
    allow[1, 0] = 1 << 3
    rows = np.array([-1] * 7 + [1, 0], np.int32)     # row 7 may only say 3, row 8 nothing
    ids = check_logits(ops, x, dict(allow=allow, allow_row=rows), torch.float32)
    assert list(ids) == [17, -1, -1, 9, 100, 7, 3000, 3, -1]
    _, logp = ops.LogitRules(allow=torch.from_numpy(allow).cuda(), allow_row=torch.from_numpy(rows).cuda()).choose(torch.from_numpy(x).cuda())
    logp = logp.cpu().numpy()
    assert logp[6] == 0 and logp[7] == 0 and abs(logp[5] + math.log(2)) < 1e-6 and logp[4] == 0


# ---------------------------------------------------------------------------
# Refusals

def _kv(**kw):
    d = dict(k=16, v=16, k_scale=16, v_scale=16, pages=4, heads=2, page=16, dim=64, format=1)
    d.update(kw)
    return _lib.Kv(**d)


def _seqs(**kw):
    d = dict(table=16, q_start=16, kv_len=16, seqs=2, table_stride=2, max_new=1, max_len=32)
    d.update(kw)
    return _lib.KvSeqs(**d)


def _rows(**kw):
    d = dict(data=16, token_stride=128, head_stride=64, tokens=0, heads=2, type=1)
    d.update(kw)
    return _lib.Rows(**d)


@pytest.mark.parametrize("kv,seqs,rows,text", [
    (dict(k=None), {}, {}, "null cache"),
    (dict(v_scale=None), {}, {}, "scales"),
    (dict(k=24), {}, {}, "16-byte"),
    (dict(k_scale=20), {}, {}, "16-byte"),
    (dict(format=2), {}, {}, "format"),
    (dict(dim=80), {}, {}, "head dim"),
    (dict(page=24), {}, {}, "page"),
    (dict(page=8), {}, {}, "page"),
    (dict(page=2048), {}, {}, "page"),
    (dict(heads=0), {}, {}, "heads"),
    (dict(pages=0), {}, {}, "pages"),
    ({}, dict(table=None), {}, "sequence"),
    ({}, dict(seqs=70000), {}, "sequences"),
    ({}, {}, dict(type=7), "type"),
    ({}, {}, dict(heads=3), "heads"),
    ({}, {}, dict(tokens=5, data=None), "null rows"),
    ({}, {}, dict(tokens=5, data=17), "aligned"),
])
def test_library_refuses(kv, seqs, rows, text):
    """Checks of arguments come before any use of the GPU, so they need none."""
    lib = _lib.load(build_if_missing=True)
    a, b, r = _kv(**kv), _seqs(**seqs), _rows(**rows)
    p = [ctypes.byref(x) for x in (a, b, r, r)]
    for call in (lambda: lib.mgb_kv_write(*p, None), lambda: lib.mgb_kv_read(*p, None), lambda: lib.mgb_kv_attend(*p, 0.125, 1, None)):
        assert call() == _lib.MGB_ERR_INVALID
        assert text in lib.mgb_last_error().decode()


def test_library_refuses_more():
    lib = _lib.load(build_if_missing=True)
    kv, seqs, r = _kv(), _seqs(), _rows()
    ref = ctypes.byref
    for args in ((None, ref(seqs), ref(r), ref(r)), (ref(kv), None, ref(r), ref(r)), (ref(kv), ref(seqs), None, ref(r)), (ref(kv), ref(seqs), ref(r), None)):
        assert lib.mgb_kv_write(*args, None) == _lib.MGB_ERR_INVALID
        assert lib.mgb_kv_attend(*args, 1.0, 0, None) == _lib.MGB_ERR_INVALID
    big = _rows(tokens=0x7fffffff)
    assert lib.mgb_kv_attend(ref(kv), ref(seqs), ref(big), ref(big), 1.0, 0, None) == _lib.MGB_ERR_INVALID
    assert lib.mgb_kv_attend(ref(kv), ref(seqs), ref(_rows(tokens=3)), ref(r), 1.0, 0, None) == _lib.MGB_ERR_INVALID
    # nothing to do is no error, and touches no memory
    assert lib.mgb_kv_write(ref(kv), ref(seqs), ref(r), ref(r), None) == _lib.MGB_OK
    assert lib.mgb_kv_attend(ref(kv), ref(_seqs(seqs=0)), ref(_rows(tokens=3)), ref(_rows(tokens=3)), 1.0, 1, None) == _lib.MGB_OK
    choose = lib.mgb_logits_choose
    assert choose(None, 0, 8, 1, 8, None, None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    assert choose(16, 3, 8, 1, 8, None, None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    assert choose(18, 0, 8, 1, 8, None, None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    assert choose(16, 0, 8, 1, 0, None, None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    assert choose(16, 0, 7, 2, 8, None, None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    assert choose(16, 0, 8, 70000, 8, None, None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    short = _lib.LogitRules(allow=16, allow_rows=1, allow_stride=1)
    assert choose(16, 0, 64, 1, 64, ref(short), None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    lost = _lib.LogitRules(bias_count=3)
    assert choose(16, 0, 64, 1, 64, ref(lost), None, None, None, 0, None) == _lib.MGB_ERR_INVALID
    assert choose(16, 0, 8, 0, 8, None, None, None, None, 0, None) == _lib.MGB_OK


def test_library_refuses_rows_written_twice():
    """A broadcast tensor as an output, whose result would be whichever store came last; as an input it is welcome."""
    lib = _lib.load(build_if_missing=True)
    ref = ctypes.byref
    kv, seqs, good = _kv(), _seqs(), _rows(tokens=3)
    for bad in (_rows(tokens=3, token_stride=0), _rows(tokens=3, head_stride=0)):
        for call in (lambda: lib.mgb_kv_read(ref(kv), ref(seqs), ref(good), ref(bad), None),
                     lambda: lib.mgb_kv_read(ref(kv), ref(seqs), ref(bad), ref(good), None),
                     lambda: lib.mgb_kv_attend(ref(kv), ref(seqs), ref(good), ref(bad), 1.0, 1, None)):
            assert call() == _lib.MGB_ERR_INVALID
            assert "overlap" in lib.mgb_last_error().decode()


@gpu_only
def test_broadcast_rows_as_inputs(ops):
    torch = _torch()
    c = Case(ops, "f16", 2, 32, 16, [5], [9])
    one = torch.randn(1, 1, 32, device="cuda").half()
    c.cache.write(c.seqs, one.expand(5, 2, 32), one.expand(5, 2, 32))
    assert torch.equal(c.cache.read(c.seqs)[0], one.expand(5, 2, 32))
    q = one.expand(5, 2, 32)
    assert torch.equal(c.cache.attend(c.seqs, q), c.cache.attend(c.seqs, q.contiguous()))
    single = torch.empty(1, 2, 32, device="cuda")[:, :, :].expand(1, 2, 32)
    assert c.cache.attend(ops.Seqs.of(c.tables, [1], c.lens), q[:1], out=single) is single


@gpu_only
def test_python_refuses(ops):
    torch = _torch()
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.PagedKV.empty(4, 2, 16, 64, "q4")
    with pytest.raises(ValueError):
        ops.PagedKV.empty(4, 2, 16, 80)
    with pytest.raises(ValueError):
        ops.PagedKV.empty(4, 2, 20, 64)
    with pytest.raises(ValueError):
        ops.PagedKV(z(4, 2, 16, 64, dtype=torch.int8), z(4, 2, 16, 64, dtype=torch.int8))
    with pytest.raises(ValueError):
        ops.PagedKV(z(4, 2, 16, 64).half(), z(4, 2, 16, 32).half())
    with pytest.raises(ValueError):
        ops.PagedKV(torch.zeros(4, 2, 16, 64).half(), torch.zeros(4, 2, 16, 64).half())
    with pytest.raises(ValueError):
        ops.Seqs(z(2, 3), z(3, **i32), z(2, **i32))
    with pytest.raises(ValueError):
        ops.Seqs(z(2, 3, **i32), z(2, **i32), z(2, **i32))
    cache, seqs = ops.PagedKV.empty(4, 2, 16, 64), ops.Seqs.of([[0], [1]], [1, 1], [3, 4])
    for q in (z(2, 4, 32), z(2, 64), z(2, 4, 64, dtype=torch.float64), z(2, 4, 128)[..., ::2], torch.zeros(2, 4, 64)):
        with pytest.raises(ValueError):
            cache.attend(seqs, q)
    with pytest.raises(ops._lib.MgbError):
        cache.attend(seqs, z(2, 3, 64))
    with pytest.raises(ops._lib.MgbError):
        cache.write(seqs, z(2, 4, 64), z(2, 4, 64))
    with pytest.raises(ops._lib.MgbError):
        cache.attend(seqs, z(2, 4, 64), out=z(3, 4, 64))
    with pytest.raises(ValueError):
        cache.read(ops.Seqs(*seqs.tensors))
    with pytest.raises(ValueError):
        ops.LogitRules(repetition=z(3))
    with pytest.raises(ValueError):
        ops.LogitRules(bias=z(3, 2))
    with pytest.raises(ValueError):
        ops.LogitRules(allow_row=z(3, **i32))
    with pytest.raises(ValueError):
        ops.LogitRules(history=z(3, 4, **i32), repetition=z(2))
    rules = ops.LogitRules(history=z(3, 4, **i32), presence=z(3))
    for x in (z(2, 100), z(3, 100, dtype=torch.float64), z(100), z(3, 200)[:, ::2]):
        with pytest.raises(ValueError):
            rules.choose(x)
    with pytest.raises(ValueError):
        rules.choose(z(3, 100), z(3, 100).half())
    with pytest.raises(ops._lib.MgbError):
        ops.LogitRules(allow=z(1, 2, **i32)).choose(z(1, 100))


# ---------------------------------------------------------------------------
# Together

@gpu_only
@pytest.mark.parametrize("fmt", ["f16", "q8"])
def test_example_serves_what_a_dense_model_says(ops, fmt):
    """examples/paged_decode.py: every token that it chose is, for a dense model in 64 bits over the same tokens, within
    the cache's rounding of the best under the rules. A row's numbers are stored to 2^-11 (f16) or 1 / 254 of its
    largest (8 bits); two layers pass that on to logits of standard deviation 1 by at most a few tenths of it."""
    import os
    import sys

    torch = _torch()
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import paged_decode as ex

    model = ex.Decoder()
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, model.vocab, (n,), generator=gen).tolist() for n in (1, 70, 33, 16)]
    bits = torch.rand(-(-model.vocab // 32), 32, generator=gen) < 0.5
    allow = (bits * torch.tensor([1 << i for i in range(31)] + [-(1 << 31)])).sum(-1).to(torch.int32).cuda()
    tokens, scores = ex.serve(model, prompts, 12, fmt, allow=allow)
    slack = 0.01 if fmt == "f16" else 0.1
    banned = (~bits.flatten()[: model.vocab]).cuda()
    for prompt, new, score in zip(prompts, tokens, scores):
        assert len(new) == 12
        seq = torch.tensor(prompt + new, device="cuda")
        x = model.start(seq, torch.arange(len(seq), device="cuda")).double()
        for layer in range(model.layers):
            q, k, v = model.project(layer, x)
            k, v = (y.repeat_interleave(model.heads // model.kv_heads, 1) for y in (k, v))
            s = torch.einsum("nhd,lhd->hnl", q, k) / model.dim ** 0.5
            s += torch.full(s.shape[1:], -math.inf, device="cuda", dtype=torch.float64).triu_(1)
            x = x + torch.einsum("hnl,lhd->nhd", s.softmax(-1), v).flatten(1) @ model.out[layer].double().T
        y = model.logits(x)
        for i, (t, logp) in enumerate(zip(new, score)):
            z = y[len(prompt) + i - 1].clone()
            said = torch.tensor(sorted(set(prompt + new[:i])), device="cuda")
            z[said] = torch.where(z[said] > 0, z[said] / 1.2, z[said] * 1.2)
            z[banned] = -math.inf
            assert not banned[t]
            assert z[t] >= z.max() - slack
            assert abs(logp - float(z[t] - z.logsumexp(0))) < slack
