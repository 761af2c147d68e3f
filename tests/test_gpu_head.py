"""GPU: the answering end (``toktier_amd.head``) against its formulas in 64
bits and, for the sampler's whole-number masses, against a model of its
definition in Python integers.

Tolerances. An e4m3 value is within half a unit of its last place: 2^-4 of
the value, or 2^-10 of the scale below e4m3's normal range. The norm's 32-bit
statistics add at most 2^-24 per addition of a chain of under 100 and four
more roundings: 1e-5 covers it.

The matrix unit aligns a group of eight products of 8-bit values to the
largest and keeps about 17 bits (a term 2^-20 below its group's largest
vanishes, measured on values chosen to show it), so a group is off by at most
8 * 2^-17 of its largest product and a result by at most 2^-14 S, S the sum of
|a w|; the 32-bit additions of groups and blocks are far below that. The
output adds half a unit of its last place: 2^-8 of the value in bf16, 2^-11 in
f16, or half of f16's least subnormal. Where the inputs are small whole
numbers nothing is dropped, and results are compared bit for bit.
"""

from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from toktier_amd import head

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
INF = math.inf


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def wide(q, scale):
    """8-bit rows as the float64 values that they stand for."""
    s = torch.exp2(scale.view(torch.uint8).double() - 127)
    return q.to(torch.float32).double() * s.repeat_interleave(128, -1)[..., :q.shape[-1]]


# ---- norm

def check_norm(x, r, w, eps, out):
    h = x.double() + (r.double() if r is not None else 0)
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()
    k = x.shape[-1]
    pad = (k + 127) // 128 * 128
    yb = torch.nn.functional.pad(y, (0, pad - k)).unflatten(-1, (-1, 128))
    amax = yb.abs().amax(-1)
    e = out.scale.view(torch.uint8).long() - 127
    s = torch.exp2(e.double())
    tiny = 1e-5
    assert bool(((amax <= 448 * s * (1 + tiny)) | (e == 127)).all())
    least = (amax > 224 * s * (1 - tiny)) | (e == -127)
    assert bool((least | ((amax == 0) & (e == 0))).all())
    got = wide(out.q, out.scale)
    per = s.repeat_interleave(128, -1)[..., :k]
    bound = torch.maximum(y.abs() * 2.0 ** -4, per * 2.0 ** -10) * (1 + tiny) + y.abs() * tiny
    assert bool(((got - y).abs() <= bound).all())
    if r is not None:
        assert torch.equal(out.residual, (x.float() + r.float()).to(x.dtype))
    # the pad of q's rows is zero
    store = torch.as_strided(out.q.view(torch.uint8), (x.numel() // k, pad), (pad, 1),
                             out.q.storage_offset())
    assert int(store[:, k:].long().sum()) == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 7), (3, 127), (2, 128), (5, 129), (1, 4096),
                                    (17, 1000), (9, 2048), (7, 2049), (33, 5001), (3, 8192),
                                    (2, 16411), (2, 65536)])
def test_norm(rows, k, dtype):
    g = gen(rows * 7 + k)
    x = (randn(g, rows, k) * 3).to(DT[dtype])
    r = (randn(g, rows, k) * 2).to(DT[dtype])
    w = (1 + 0.3 * randn(g, k)).to(DT[dtype])
    check_norm(x, r, w, 1e-6, head.rms_norm_fp8(x, w, residual=r))
    out = head.rms_norm_fp8(x, w.float(), eps=1e-3)
    assert out.residual is None
    check_norm(x, None, w.float(), 1e-3, out)


def test_norm_strides_axes_and_the_sum_in_place():
    g = gen(3)
    big = randn(g, 6, 3, 400).to(torch.bfloat16)
    x, w = big[:, :, 3:260], (1 + 0.2 * randn(g, 257)).to(torch.bfloat16)
    with pytest.raises(ValueError, match="stride"):
        head.rms_norm_fp8(big[:, :2, :257], w)
    r = randn(g, 6, 3, 257).to(torch.bfloat16)
    want = head.rms_norm_fp8(x.contiguous(), w, residual=r)
    keep = r.clone()
    got = head.rms_norm_fp8(x, w, residual=r, residual_out=r)
    assert got.residual is r
    for a, b in ((got.q.view(torch.uint8), want.q.view(torch.uint8)),
                 (got.scale.view(torch.uint8), want.scale.view(torch.uint8)),
                 (r, want.residual)):
        assert torch.equal(a, b)
    check_norm(x.reshape(18, 257), keep.view(18, 257), w, 1e-6,
               head.rms_norm_fp8(x, w, residual=keep)._replace(
                   q=got.q.flatten(0, 1), scale=got.scale.flatten(0, 1),
                   residual=got.residual.view(18, 257)))
    # one row for all: stride 0
    one = randn(g, 1, 512).expand(5, 512)
    out = head.rms_norm_fp8(one, torch.ones(512, device="cuda"))
    check_norm(one.contiguous(), None, torch.ones(512, device="cuda"), 1e-6, out)
    assert head.rms_norm_fp8(x[:0], w).q.shape == (0, 3, 257)


def test_norm_zeros_extremes_and_what_is_not_finite():
    one = torch.ones(384, device="cuda")
    x = torch.zeros(6, 384, device="cuda")
    x[1, :128] = 1e-30          # below the smallest scale after the norm: 0 or subnormal
    x[1, 128:] = 1.0
    x[2] = 1e18                 # each square is below float32's largest, their sum is not
    x[3, 5] = INF
    x[4, 5] = math.nan
    out = head.rms_norm_fp8(x, one)
    assert bool((wide(out.q, out.scale)[0] == 0).all())
    assert out.scale.view(torch.uint8)[0].tolist() == [127] * 3  # zeros: a scale of 1
    check_norm(x[1:3], None, one, 1e-6, out._replace(q=out.q[1:3], scale=out.scale[1:3]))
    got = wide(out.q, out.scale)
    assert bool(got[3, 5].isnan()) and bool(got[4].isnan().all())
    assert bool((got[3].nan_to_num(0) == 0).all())  # the others over an infinite root
    # powers of two at a scale's edge: 448 fits, the next value does not
    edge = torch.full((1, 128), 448.0, device="cuda")
    w = torch.full((128,), 448.0, device="cuda")
    out = head.rms_norm_fp8(edge, w, eps=0.0)
    assert out.scale.view(torch.uint8).tolist() == [[127]]
    assert bool((out.q.float() == 448).all())


# ---- product

def quantized(g, rows, k, spread=1.0):
    x = randn(g, rows, k) * torch.exp(spread * randn(g, rows, 1))
    return head.quantize_fp8(x)


def check_matmul(a, w, out, dtype, got):
    a, w = wide(*a), wide(*w)
    want, size = a @ w.t(), a.abs() @ w.abs().t()
    bound = 2.0 ** -14 * size + want.abs() * HALF_UNIT[dtype]
    if dtype == "f16":
        bound += 2.0 ** -25
    assert got.dtype == DT[dtype] and got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), f"over by {float(off.max())}"


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 100, 129, 200, 257, 300])
@pytest.mark.parametrize("n,k,dtype", [(1, 1, "bf16"), (40, 100, "f16"), (257, 128, "bf16"),
                                       (515, 1000, "f16"), (1000, 1111, "bf16"),
                                       (513, 2048, "f16"), (300, 4096, "bf16"),
                                       (129, 8192, "bf16"), (77, 9000, "bf16")])
def test_matmul(m, n, k, dtype):
    g = gen(m * 31 + n + k)
    a, w = quantized(g, m, k, 0.5), quantized(g, n, k, 0.5)
    if dtype == "f16":
        w = (w[0], (w[1].view(torch.uint8) - 4).view(torch.float8_e8m0fnu))
    check_matmul(a, w, None, dtype, head.matmul_fp8(*a, *w, out_dtype=DT[dtype]))


@pytest.mark.parametrize("m", [1, 5, 16, 17, 40, 64, 65, 128, 190, 256, 500])
@pytest.mark.parametrize("n,k", [(1, 16), (33, 130), (600, 384), (1025, 513), (333, 1152),
                                 (200, 4224), (64, 8320), (31, 12345)])
def test_matmul_of_whole_numbers_is_exact(m, n, k):
    """Values -2 .. 2 in blocks scaled by 1, 2, 4 and 8: sums of whole numbers
    below 2^24, of which f16's largest values hold 2048 exactly (the output
    is compared with the exact sum rounded once)."""
    g = gen(m + n + k)
    blocks = (k + 127) // 128

    def whole(rows):
        pad = torch.zeros(rows, blocks * 128, device="cuda")
        pad[:, :k] = torch.randint(-2, 3, (rows, k), generator=g, device="cuda")
        scale = torch.randint(127, 131, (rows, blocks), generator=g, device="cuda")
        return (pad.to(torch.float8_e4m3fn)[:, :k],
                scale.to(torch.uint8).view(torch.float8_e8m0fnu))

    a, w = whole(m), whole(n)
    got = head.matmul_fp8(*a, *w, out_dtype=torch.bfloat16)
    want = wide(*a) @ wide(*w).t()
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(got, want.float().to(torch.bfloat16))


@pytest.mark.parametrize("m", [1, 3, 16, 30, 64])
@pytest.mark.parametrize("n,k", [(333, 1024), (97, 2048), (2500, 2048), (130, 4096), (1000, 4100),
                                 (9000, 5000), (77, 6144), (5001, 6144), (50, 6145), (600, 8192)])
def test_matmul_of_whole_numbers_where_k_fills_the_waves_or_not(m, n, k):
    """8 or 16 waves share k: all of them full, the last in part, some empty."""
    test_matmul_of_whole_numbers_is_exact(m, n, k)


@pytest.mark.parametrize("m", [66, 96, 130, 192, 257, 320, 321, 449, 777])
@pytest.mark.parametrize("n,k", [(300, 100), (257, 128), (1000, 640), (513, 1100), (70, 5200)])
def test_matmul_of_whole_numbers_where_a_tile_ends_in_any_wave(m, n, k):
    """The last tile has rows for one wave, some of them or all."""
    test_matmul_of_whole_numbers_is_exact(m, n, k)


@pytest.mark.parametrize("far", ["a", "w", "scales"])
@pytest.mark.parametrize("m", [2, 9, 21])
def test_matmul_of_rows_far_apart(m, far):
    """Rows 8 MB apart: what is added up 32 bits of offset does not hold."""
    g = gen(m)
    n, k, step = 300 if far == "w" else 130, 8200, 1 << 23
    a, w = quantized(g, m, k, 0.5), quantized(g, n, k, 0.5)

    def apart(t, stride):
        at = torch.zeros(t.shape[0] * stride, dtype=torch.uint8, device="cuda").as_strided(
            (t.shape[0], t.shape[1]), (stride, 1))
        at.copy_(t.view(torch.uint8))
        return at.view(t.dtype)

    fa, fw = a, w
    if far == "a":
        fa = (apart(a[0], step), a[1])
    elif far == "w":
        fw = (apart(w[0], step), w[1])
    else:
        fa, fw = (a[0], apart(a[1], step)), (w[0], apart(w[1], step))
    check_matmul(a, w, None, "bf16", head.matmul_fp8(*fa, *fw, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("n", [50257, 30000])
def test_matmul_over_a_vocabulary(m, n):
    g = gen(m + n)
    a, w = quantized(g, m, 640), quantized(g, n, 640)
    check_matmul(a, w, None, "bf16", head.matmul_fp8(*a, *w, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_matmul_reads_nothing_beyond_k_and_writes_nothing_beyond_n(m):
    """Rows in wider storage: NaN behind k, other values behind n."""
    g = gen(m)
    k, n = 1000, 300
    aq, asc = quantized(g, m, k)
    wq, wsc = quantized(g, n, k)
    a = torch.full((m, 1040), 0x7f, dtype=torch.uint8, device="cuda")
    w = torch.full((n, 1072), 0x7f, dtype=torch.uint8, device="cuda")
    a[:, :k], w[:, :k] = aq.view(torch.uint8), wq.view(torch.uint8)
    scales = torch.full((n, 11), 255, dtype=torch.uint8, device="cuda")
    scales[:, :8] = wsc.view(torch.uint8)
    out = torch.full((m, n + 9), 7.0, device="cuda", dtype=torch.bfloat16)
    fp8 = torch.float8_e4m3fn
    got = head.matmul_fp8(a.view(fp8)[:, :k], asc, w.view(fp8)[:, :k], scales[:, :8],
                          out=out[:, 4:n + 4])
    check_matmul((aq, asc), (wq, wsc), None, "bf16", got)
    assert bool((out[:, :4] == 7).all()) and bool((out[:, n + 4:] == 7).all())


def test_matmul_scales_far_apart_nan_scales_and_axes():
    g = gen(9)
    a, w = quantized(g, 6, 512), quantized(g, 50, 512)
    sa, sw = a[1].view(torch.uint8).clone(), w[1].view(torch.uint8).clone()
    sa[:, 1] -= 60
    sa[:, 2] += 40
    sw[:, 1] += 61
    sw[:, 2] -= 39
    a, w = (a[0], sa.view(torch.float8_e8m0fnu)), (w[0], sw.view(torch.float8_e8m0fnu))
    got = head.matmul_fp8(*a, *w, out_dtype=torch.bfloat16)
    check_matmul(a, w, None, "bf16", got)
    three = head.matmul_fp8(a[0].view(2, 3, 512), a[1].view(2, 3, 4), *w, out_dtype=torch.bfloat16)
    assert torch.equal(three, got.view(2, 3, 50))
    sw[7, 3] = 255
    got = head.matmul_fp8(*a, w[0], sw, out_dtype=torch.bfloat16)
    assert bool(got[:, 7].isnan().all()) and not bool(got[:, :7].isnan().any())
    assert head.matmul_fp8(a[0][:0], a[1][:0], *w).shape == (0, 50)


def test_matmul_of_a_row_is_the_same_beside_others():
    """A row's sums do not depend on the other rows of a batch of 5 to 16."""
    g = gen(4)
    a, w = quantized(g, 16, 2048), quantized(g, 1000, 2048)
    all_ = head.matmul_fp8(*a, *w)
    for rows in (slice(0, 5), slice(9, 16)):
        some = head.matmul_fp8(a[0][rows], a[1][rows], *w)
        assert torch.equal(some, all_[rows])


# ---- sampler

def model(x, u, t, k, p, floor, allowed):
    """The definition for one row, in Python integers over the row's weights
    (float32, from torch's elementary operations on the device)."""
    x = x.float()
    ok = x > -INF
    if allowed is not None:
        bits = allowed.cpu().numpy().view(np.uint32)
        i = np.arange(x.shape[0])
        ok &= torch.tensor((bits[i // 32] >> (i % 32)) & 1 != 0, device=x.device)
    if not bool(ok.any()):
        return -1, -INF
    x = torch.where(ok, x, -INF)
    greedy = not t > 0
    one = torch.ones((), device=x.device)
    step = (one * math.log2(math.e)) / (one if greedy else one * t)
    top = x.max()
    w = torch.where(x == top, 1.0, torch.exp2((x - top) * step))
    w = torch.where(ok, w, 0.0)
    q = [int(v) for v in (w * 2.0 ** 40).to(torch.int64).tolist()]
    xs, ws, okl = x.tolist(), w.tolist(), ok.tolist()
    order = sorted((i for i in range(len(xs)) if okl[i]), key=lambda i: (-xs[i], i))
    if greedy:
        k = 1
    if k > 0:
        order = order[:k]
    p32 = float(np.float32(p))
    if p32 < 1:
        part = max(1, math.ceil(p32 * float(sum(q[i] for i in order))))
        kept, before = [], 0
        for i in order:
            if before >= part:
                break
            kept.append(i)
            before += q[i]
        order = kept
    order = sorted(i for i in order if ws[i] >= float(np.float32(floor)))
    total = sum(q[i] for i in order)
    at = min(max(0, math.floor(float(np.float32(u)) * float(total))), total - 1)
    for i in order:
        if at < q[i]:
            return i, math.log(Fraction(q[i], total))
        at -= q[i]
    raise AssertionError


def rows_of(kind, rows, vocab, dtype, seed):
    g = gen(seed)
    x = randn(g, rows, vocab)
    if kind == "zipf":
        x = -1.5 * torch.rand(rows, vocab, generator=g, device="cuda").clamp_(min=1e-9).log() + 0.3 * x
    elif kind == "flat":
        x = 0.01 * x
    elif kind == "equal":
        x = torch.zeros_like(x)
    elif kind == "steps":      # many equal logits
        x = (2 * x).round()
    elif kind == "sharp":
        x = 30 * x
    elif kind == "lowest":     # masks written as the type's lowest value
        x = torch.where(torch.rand(rows, vocab, generator=g, device="cuda") < 0.9,
                        torch.finfo(DT[dtype]).min, x)
    return x.to(DT[dtype])


def check_rows(x, u, allowed=None, **settings):
    got = head.sample(x, u, allowed=allowed, **settings)
    rows = x.shape[0]

    def of(name, r, default):
        v = settings.get(name, default)
        return float(v[r]) if isinstance(v, torch.Tensor) else v

    for r in range(rows):
        mask = None if allowed is None else allowed[r if allowed.shape[0] > 1 else 0]
        want, lp = model(x[r], float(u[r]), of("temperature", r, 1.0), int(of("top_k", r, 0)),
                         of("top_p", r, 1.0), of("min_p", r, 0.0), mask)
        assert int(got.ids[r]) == want, (r, settings)
        # two conversions, a quotient and a logarithm in 32 bits, on a share or on
        # what is missing to one
        have = float(got.logprob[r])
        assert have == lp or abs(have - lp) <= 4e-7 * max(1.0, abs(lp)), (r, have, lp)
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.6, top_k=1), dict(top_k=5),
            dict(temperature=1.3, top_k=50, top_p=0.9), dict(top_p=0.5), dict(top_p=0.95),
            dict(top_p=0.999, temperature=1.5), dict(min_p=0.1), dict(min_p=1.0),
            dict(top_p=0.9, min_p=0.02), dict(top_k=700, top_p=0.99, min_p=0.001),
            dict(top_p=0.0), dict(temperature=0.05), dict(temperature=50.0, top_k=3000)]


@pytest.mark.parametrize("kind", ["normal", "zipf", "flat", "equal", "steps", "sharp", "lowest"])
@pytest.mark.parametrize("vocab,dtype", [(1, "f32"), (2, "bf16"), (33, "f16"), (1000, "f32"),
                                         (1031, "bf16"), (5003, "f32"), (20011, "bf16")])
def test_sample(kind, vocab, dtype):
    x = rows_of(kind, 2, vocab, dtype, vocab)
    g = gen(vocab + 1)
    for settings in SETTINGS:
        check_rows(x, torch.rand(2, generator=g, device="cuda"), **settings)


@pytest.mark.parametrize("kind", ["normal", "zipf", "flat", "steps"])
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 151669, "f32"), (3, 50257, "bf16"),
                                              (1, 200019, "f16")])
def test_sample_over_a_vocabulary(kind, rows, vocab, dtype):
    x = rows_of(kind, rows, vocab, dtype, vocab)
    g = gen(vocab + 1)
    for settings in SETTINGS[:1] + SETTINGS[4:12]:
        check_rows(x, torch.rand(rows, generator=g, device="cuda"), **settings)


def test_sample_settings_of_each_row_and_its_mask():
    g = gen(11)
    rows, vocab = 300, 3001
    x = rows_of("zipf", rows, vocab, "bf16", 5)
    pick = lambda values, dt: torch.tensor(values, device="cuda", dtype=dt)[  # noqa: E731
        torch.randint(0, len(values), (rows,), generator=g, device="cuda")]
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g,
                            device="cuda").to(torch.int32)
    allowed[7] = 0                # a row that its mask leaves empty
    allowed[8] = 0
    allowed[8, 93] = 1 << 24      # token 3000, the last, alone
    got = check_rows(x, torch.rand(rows, generator=g, device="cuda"), allowed,
                     temperature=pick([0.0, -1.0, 0.7, 1.0, 2.0], torch.float32),
                     top_k=pick([0, -3, 1, 40, 900, 10 ** 9], torch.int32),
                     top_p=pick([1.0, 0.9, 0.3, 2.0, -1.0], torch.float32),
                     min_p=pick([0.0, 0.05, -1.0], torch.float32))
    assert int(got.ids[7]) == -1 and float(got.logprob[7]) == -INF
    assert int(got.ids[8]) == 3000 and float(got.logprob[8]) == 0.0
    # one mask for all rows
    check_rows(x[:20], torch.rand(20, generator=g, device="cuda"), allowed[9:10], top_p=0.8)


def test_sample_infinities_nan_and_the_ends_of_u():
    x = torch.full((8, 700), -INF, device="cuda")
    x[1] = math.nan
    x[2, 5] = -2.0
    x[3, [4, 9]] = INF
    x[3, 20:40] = 3.0
    x[4, :] = torch.finfo(torch.float32).min
    x[5, 699] = torch.finfo(torch.float32).max
    x[5, 0] = torch.finfo(torch.float32).min
    x[6, 10], x[6, 600] = -0.0, 0.0     # equal: the lower index first
    x[7, 3:9] = math.nan
    x[7, 100:110] = 1.0
    for u in (0.0, 0.25, 0.5, float(np.nextafter(np.float32(1), np.float32(0)))):
        us = torch.full((8,), u, device="cuda")
        for settings in (dict(), dict(top_k=1), dict(top_p=0.6), dict(temperature=0.0),
                         dict(temperature=1e-30), dict(temperature=1e30), dict(min_p=0.5)):
            check_rows(x, us, **settings)
    got = head.sample(x, torch.zeros(8, device="cuda"))
    assert got.ids.tolist() == [-1, -1, 5, 4, 0, 699, 10, 100]
    # u outside [0, 1) draws the first or the last that stays
    for u, want in ((-3.0, 4), (1.0, 9), (7.0, 9), (math.nan, 4)):
        assert int(head.sample(x[3:4], torch.tensor([u], device="cuda")).ids) == want


def test_sample_rows_in_wider_storage_and_of_one_stride():
    g = gen(2)
    store = torch.full((5, 4100), 1e30, device="cuda")
    store[:, 3:4004] = randn(g, 5, 4001)
    u = torch.rand(5, generator=g, device="cuda")
    check_rows(store[:, 3:4004], u, top_p=0.9)
    check_rows(store[:1, 3:4004].expand(5, 4001), u, top_k=20)
    assert head.sample(store[:0], u[:0]).ids.shape == (0,)


def test_sample_gives_a_row_the_same_token_in_any_batch():
    g = gen(21)
    x = rows_of("zipf", 600, 60007, "f32", 3)
    u = torch.rand(600, generator=g, device="cuda")
    for settings in (dict(top_p=0.95), dict(), dict(top_k=40), dict(temperature=1.5, top_p=0.99)):
        all_ = head.sample(x, u, **settings)
        for cut in (slice(0, 1), slice(5, 9), slice(100, 160), slice(300, 600)):
            part = head.sample(x[cut], u[cut], **settings)
            assert torch.equal(part.ids, all_.ids[cut])
            assert torch.equal(part.logprob, all_.logprob[cut])


def test_sample_draws_by_the_weights():
    """4,096 draws at evenly spaced u of one row: each token's count is its
    share of them, to one."""
    g = gen(8)
    x = randn(g, 1, 500)
    n = 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = head.sample(x.expand(n, 500), u, temperature=0.8)
    share = torch.softmax(x[0].double() / 0.8, 0) * n
    count = torch.bincount(got.ids.long(), minlength=500).double()
    assert float((count - share).abs().max()) <= 1.01


# ---- together

def test_output_head_on_a_stream_and_in_a_graph():
    g = gen(30)
    k, n, vocab, rows = 512, 2304, 2300, 12
    hidden, res = randn(g, rows, k).bfloat16(), randn(g, rows, k).bfloat16()
    out = head.OutputHead((1 + 0.1 * randn(g, k)).bfloat16(), *head.quantize_fp8(randn(g, n, k)),
                          vocab=vocab)
    u = torch.rand(rows, generator=g, device="cuda")
    y = head.rms_norm_fp8(hidden, out.norm_weight, residual=res)
    logits = head.matmul_fp8(y.q, y.scale, out.w, out.w_scale)
    want = head.sample(logits, u, temperature=0.7, top_p=0.9)
    assert logits.shape == (rows, vocab) and int(want.ids.max()) < vocab
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = out.next_ids(hidden, u, residual=res, temperature=0.7, top_p=0.9)
    side.synchronize()
    assert torch.equal(got.ids, want.ids) and torch.equal(got.logprob, want.logprob)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = out.next_ids(hidden, u, residual=res, temperature=0.7, top_p=0.9)
    for step in range(4):
        u.copy_(torch.rand(rows, generator=g, device="cuda"))
        hidden.copy_(randn(g, rows, k).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        eager = out.next_ids(hidden, u, residual=res, temperature=0.7, top_p=0.9)
        assert torch.equal(held.ids, eager.ids) and torch.equal(held.logprob, eager.logprob)


def test_sample_at_a_temperature_whose_inverse_is_infinite():
    """Below 4.3e-39 log2(e) / T is infinite: the largest logits weigh 1, all
    others nothing."""
    x = randn(gen(41), 4, 3000)
    x[1, 700], x[1, 2000] = 9.0, 9.0
    x[2, 5:9] = -INF
    x[3, 2999] = INF
    for u in (0.0, 0.4, 0.6):
        us = torch.full((4,), u, device="cuda")
        for settings in (dict(), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=40),
                         dict(top_k=1500, top_p=0.5)):
            check_rows(x, us, temperature=1e-40, **settings)
            check_rows(x, us, temperature=torch.full((4,), 1e-40, device="cuda"), **settings)


def test_sample_the_widest_row_of_equal_logits():
    """Their masses sum to just below 2**64; the tokens before the one drawn
    are exactly floor(u * how many stay)."""
    v = 2 ** 24 - 1
    x = torch.zeros(1, v, dtype=torch.bfloat16, device="cuda")
    top = float(np.nextafter(np.float32(1), np.float32(0)))
    for u in (0.0, 0.3, 0.75, top):
        us = torch.tensor([u], device="cuda")
        u = float(us)
        assert int(head.sample(x, us).ids) == math.floor(u * float(v * 2 ** 40)) >> 40
        half = (v + 1) // 2
        got = head.sample(x, us, top_p=0.5)
        assert int(got.ids) == math.floor(u * half)
        assert float(got.logprob) == pytest.approx(-math.log(half), rel=1e-6)


def test_example_from_text_to_text():
    """examples/next_token.py: the same seed answers the same, in the
    family's own tokens, none of them an added one."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "next_token.py"
    spec = importlib.util.spec_from_file_location("next_token", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    first = example.main("gpt2", steps=5, hidden=256, seed=3)
    assert len(first) == len(example.PROMPTS) and all(first)
    assert "<|endoftext|>" not in "".join(first)
    assert example.main("gpt2", steps=5, hidden=256, seed=3) == first
    assert example.main("gpt2", steps=5, hidden=256, seed=4) != first


def test_refusals_on_the_device():
    x = torch.zeros(2, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    q, s = head.quantize_fp8(torch.ones(4, 256, device="cuda"))
    with pytest.raises(TypeError, match="float64"):
        head.rms_norm_fp8(x.double(), w)
    with pytest.raises(ValueError, match="weight"):
        head.rms_norm_fp8(x, w[:255])
    with pytest.raises(TypeError, match="weight"):
        head.rms_norm_fp8(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        head.rms_norm_fp8(x, w, residual=x[:1])
    with pytest.raises(ValueError, match="dense"):
        head.rms_norm_fp8(x.t().contiguous().t(), w)
    with pytest.raises(head.EngineError, match="TK_E_UNSUPPORTED"):
        head.rms_norm_fp8(torch.zeros(1, 65537, device="cuda"), torch.ones(65537, device="cuda"))
    with pytest.raises(TypeError, match="wanted"):
        head.matmul_fp8(x, s, q, s)
    with pytest.raises(ValueError, match="scale"):
        head.matmul_fp8(q, s[:, :1], q, s)
    with pytest.raises(ValueError, match="rows of"):
        head.matmul_fp8(q[:, :128], s[:, :1], q, s)
    with pytest.raises(head.EngineError, match="aligned"):
        head.matmul_fp8(q[:, 4:132], s[:, :1], q[:, :128], s[:, :1])
    u = torch.zeros(2, device="cuda")
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1),
                dict(top_p=1.5), dict(min_p=-0.1), dict(top_k=torch.zeros(2, device="cuda")),
                dict(top_p=torch.zeros(3, device="cuda")),
                dict(allowed=torch.zeros(2, 7, device="cuda", dtype=torch.int32))):
        with pytest.raises(ValueError):
            head.sample(x, u, **bad)
    with pytest.raises(ValueError, match="u is"):
        head.sample(x, u[:1])
    with pytest.raises(ValueError, match="on cpu"):
        head.sample(x, u.cpu())


@pytest.mark.parametrize("k", [1000, 1111, 4104, 6144])
def test_matmul_of_a_single_row_of_any_stride(k):
    """A contiguous row whose length is no multiple of 16, as a and as w."""
    g = gen(k)
    one, many = quantized(g, 1, k), quantized(g, 90, k)
    tight = torch.empty(1, k, dtype=torch.uint8, device="cuda")
    tight.copy_(one[0].view(torch.uint8))
    tight = tight.view(torch.float8_e4m3fn)
    assert tight.stride(0) == k
    assert torch.equal(head.matmul_fp8(tight, one[1], *many), head.matmul_fp8(*one, *many))
    assert torch.equal(head.matmul_fp8(*many, tight, one[1]), head.matmul_fp8(*many, *one))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k", [1, 256, 1000, 5001])
def test_one_axis_is_one_row(k, dtype):
    """``[k]`` gives what ``[1, k]`` gives, the sum in place among it."""
    g = gen(k)
    x, r = randn(g, k).to(DT[dtype]), randn(g, k).to(DT[dtype])
    norm_w, w = (1 + 0.2 * randn(g, k)).to(DT[dtype]), quantized(g, 77, k)
    want = head.rms_norm_fp8(x[None], norm_w, residual=r[None])
    keep = r.clone()
    got = head.rms_norm_fp8(x, norm_w, residual=r, residual_out=r)
    assert got.residual is r and got.q.shape == (k,)
    for a, b in ((got.q.view(torch.uint8), want.q.view(torch.uint8)),
                 (got.scale.view(torch.uint8), want.scale.view(torch.uint8)),
                 (r, want.residual)):
        assert torch.equal(a, b[0])
    c = head.matmul_fp8(want.q, want.scale, *w)
    assert torch.equal(head.matmul_fp8(got.q, got.scale, *w), c[0])
    assert torch.equal(head.OutputHead(norm_w, *w).logits(x, residual=keep), c[0])


def test_inputs_that_require_grad_give_the_same_and_no_gradient():
    g = gen(51)
    x, r, w = randn(g, 4, 300), randn(g, 4, 300), 1 + 0.2 * randn(g, 300)
    out = head.OutputHead(w, *head.quantize_fp8(randn(g, 77, 300)))
    u = torch.rand(4, generator=g, device="cuda")
    want = head.rms_norm_fp8(x, w, residual=r)
    ids = out.next_ids(x, u, residual=r)
    x.requires_grad_(True)
    got = head.rms_norm_fp8(x, w, residual=r)
    assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8))
    assert torch.equal(got.scale.view(torch.uint8), want.scale.view(torch.uint8))
    assert torch.equal(got.residual, want.residual)
    with pytest.raises(NotImplementedError, match="rms_norm_fp8"):
        got.residual.sum().backward()
    drawn = out.next_ids(x, u, residual=r)
    assert torch.equal(drawn.ids, ids.ids) and torch.equal(drawn.logprob, ids.logprob)
    with pytest.raises(NotImplementedError, match="sample"):
        drawn.logprob.sum().backward()
    assert x.grad is None
    with pytest.raises(ValueError, match="residual_out"):
        head.rms_norm_fp8(x, w, residual=r, residual_out=r)


@pytest.mark.parametrize("k", [1, 128, 1000, 5001, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size,eps", [(1e19, 1e-6), (3e21, 1e-6), (5e30, 0.0), (3e38, 1e-6), (3e38, 3e38),
                                      (1e-18, 0.0), (1e-25, 0.0), (1e-25, 1e-30), (1e-39, 0.0),
                                      (1e-25, 1e-6), (1e-12, 5e-20)])
def test_norm_of_rows_whose_squares_leave_32_bits(k, dtype, size, eps):
    """Finite rows have finite norms: squares above 2^128 or below 2^-126."""
    g = gen(k)
    x = (size * (1 - 2 * torch.rand(4, k, generator=g, device="cuda", dtype=torch.float64))).to(DT[dtype])
    x[1, k // 2:] *= 1e-3
    x[2] = size
    w = (1 + 0.2 * randn(g, k)).to(DT[dtype])
    out = head.rms_norm_fp8(x, w, eps=eps)
    # a row that the thousandth leaves at zero is 0 / 0 where eps is 0
    none = (x == 0).all(-1) & (eps == 0)
    assert bool(out.q[none].float().isnan().all())
    for r in torch.nonzero(~none).flatten().tolist():
        cut = slice(r, r + 1)
        check_norm(x[cut], None, w, eps, out._replace(q=out.q[cut], scale=out.scale[cut]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_whose_output_is_infinite_is_nan_there(dtype):
    """Infinite weights and products beyond 32 bits: NaN in their places, which
    the scale of their block does not count."""
    k = 512
    x = torch.ones(2, k, device="cuda", dtype=DT[dtype])
    w = torch.ones(k, device="cuda", dtype=DT[dtype])
    w[3], w[130], w[131], w[300] = INF, -INF, math.nan, INF
    out = head.rms_norm_fp8(x, w, eps=0.0)
    got = wide(out.q, out.scale)
    bad = torch.zeros(2, k, dtype=torch.bool, device="cuda")
    bad[:, [3, 130, 131, 300]] = True
    assert torch.equal(got.isnan(), bad)
    assert bool((got[~bad] == 1).all())
    assert out.scale.view(torch.uint8).tolist() == [[127 - 8] * 4] * 2  # 1 is 256 * 2^-8
    # one value of a row of zeros is sqrt(k) = 22 after the norm
    x = torch.zeros(2, k, device="cuda", dtype=DT[dtype])
    x[:, 200] = 2.0
    w = torch.ones(k, device="cuda", dtype=DT[dtype])
    w[200] = torch.finfo(DT[dtype]).max
    out = head.rms_norm_fp8(x, w)
    got = wide(out.q, out.scale)
    assert bool(got[:, 200].isnan().all()) and float(got.nan_to_num(0).abs().sum()) == 0


@pytest.mark.parametrize("k", [257, 1000, 4096])
def test_norm_writes_the_sum_into_a_strided_view(k):
    g = gen(k)
    x, r = randn(g, 7, k).bfloat16(), randn(g, 7, k).bfloat16()
    w = (1 + 0.2 * randn(g, k)).bfloat16()
    store = torch.full((7, k + 21), 5.0, device="cuda", dtype=torch.bfloat16)
    view = store[:, 9:9 + k]
    out = head.rms_norm_fp8(x, w, residual=r, residual_out=view)
    assert out.residual is view
    check_norm(x, r, w, 1e-6, out)
    assert bool((store[:, :9] == 5).all()) and bool((store[:, 9 + k:] == 5).all())
    view.copy_(r)
    again = head.rms_norm_fp8(x, w, residual=view, residual_out=view)
    assert torch.equal(again.residual, out.residual)
    assert torch.equal(again.q.view(torch.uint8), out.q.view(torch.uint8))


@pytest.mark.parametrize("rows,vocab,kind,settings", [
    (40, 20011, "normal", dict(top_p=0.95)), (33, 20011, "normal", dict(top_p=0.99, temperature=1.5)),
    (70, 9001, "normal", dict(top_p=0.97, min_p=0.01)), (300, 5003, "normal", dict(top_p=0.95)),
    (70, 5003, "steps", dict(top_p=0.98, temperature=2.0)), (270, 5003, "flat", dict(top_p=0.9))])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_more_wide_rows_than_a_turn_takes(rows, vocab, kind, settings, dtype):
    """Sets of over 2,048 tokens in more rows than 32, or 256."""
    x = rows_of(kind, rows, vocab, dtype, rows)
    share = torch.softmax(x.double() / settings.get("temperature", 1.0), -1).sort(descending=True).values
    kept = (share.cumsum(-1) - share < settings["top_p"]).sum(-1)
    assert int((kept > 2048).sum()) > (256 if rows > 256 else 32) or "min_p" in settings
    check_rows(x, torch.rand(rows, generator=gen(rows), device="cuda"), **settings)


def test_a_refused_device_leaves_no_error_behind():
    """A failed query's error would be raised by the next check of a launch,
    torch's among them."""
    p = 1 << 20  # an address that no call reads
    lib = head.lib()
    torch.zeros(1, device="cuda")
    norm = [p, 0, p, p, p, 0, 4, 256, 256, 0, 256, 2, 0, 1e-6, 0, 0, 63]
    assert lib.tk_head_norm(head._NORM.pack(*norm), None) == -3
    assert lib.hipPeekAtLastError() == 0
    assert float(torch.ones(3, device="cuda").sum()) == 3


@pytest.mark.parametrize("m", [1, 20, 140])
@pytest.mark.parametrize("n,k", [(130, 128), (97, 1000), (200, 2048), (90, 4096)])
@pytest.mark.parametrize("spread", ["one large", "heavy tails"])
def test_matmul_of_unequal_products_keeps_the_stated_bound(m, n, k, spread):
    """The unit adds the products of 8 neighbours along k cut to multiples of
    2^-13 of the power of two that the exponents of the largest one's factors
    make, so 7 products lose less than 7 * 2^-13 of the largest; groups and
    blocks add up in 32 bits, k / 8 + 32 additions of at most 2^-24 of the sum
    of |a w| each. With one large product in each group the others lie below
    that cut."""
    g = gen(m + n + k)
    if spread == "one large":
        x = torch.full((m, k), 0.03, device="cuda")
        y = torch.full((n, k), 1.0, device="cuda")
        x[:, ::8], y[:, ::8] = 16.0, 16.0
    else:
        x = randn(g, m, k) * torch.exp(2 * randn(g, m, k))
        y = randn(g, n, k) * torch.exp(2 * randn(g, n, k))
    a, w = head.quantize_fp8(x), head.quantize_fp8(y)
    A, W = wide(*a), wide(*w)
    pad = (0, -k % 8)
    ga = torch.nn.functional.pad(A.abs(), pad).unflatten(1, (-1, 8))
    gw = torch.nn.functional.pad(W.abs(), pad).unflatten(1, (-1, 8))
    largest = sum((ga[:, None, b] * gw[None, :, b]).amax(-1) for b in range(ga.shape[1]))
    want, size = A @ W.t(), A.abs() @ W.abs().t()
    bound = 7 * 2.0 ** -13 * largest + (k / 8 + 32) * 2.0 ** -24 * size + want.abs() * 2.0 ** -8
    off = (head.matmul_fp8(*a, *w).double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
