"""GPU: the draw from logits (st_sample_logits) and the product with 4-bit weights (st_gemm_q4) against plain 64-bit
implementations, one by one and in a row.

Tolerances.  Token ids are exact: masks and draws are whole-number sums, and no test puts a border within 2^-40 of a draw by
chance.  logp is one rounding to f32 (2^-24 of the value) of a logarithm whose argument is good to 1e-12.  A product is
y (1 + r) + d: r the one rounding to y's type (half a step: 2^-24, 2^-8, 2^-11), |d| <= ((K + 64) 2^-24 + 2^-22) A + 2^-39 K max|x| max|w|
with A = sum |x| |w|: f32 additions of K terms and of the joins, the 22 bits that an f32 x keeps, and what its row's power of
two takes from values far below the row's largest."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda", 0)


# ---- the draw ---------------------------------------------------------------------------------------------------------

def plain_sample(row, u, temperature, top_k, top_p, min_p):
    """the definition, on one row in 64 bits (settings as the 32 bits that the kernel is given)"""
    row = row.astype(np.float64)
    row = np.where(np.isnan(row), -np.inf, row)
    order = np.argsort(-row, kind="stable")
    order = order[:int((row > -np.inf).sum())]
    if len(order) == 0:
        return -1, -np.inf
    top = row[order[0]]
    if not temperature > 0:
        return int(order[0]), 0.0
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.where(row[order] == top, 1.0, np.exp((row[order] - top) / np.float64(np.float32(temperature))))
    c = np.cumsum(w)
    keep = len(order)
    if top_p < 1:
        keep = int(np.searchsorted(np.concatenate(([0.0], c))[:-1], np.float64(np.float32(top_p)) * c[-1], side="left"))
    if min_p > 0:
        keep = min(keep, int((w >= np.float64(np.float32(min_p))).sum()))
    keep = max(keep, 1)
    at = min(int(np.searchsorted(c[:keep], np.float64(u) * c[keep - 1], side="right")), keep - 1)
    return int(order[at]), math.log(w[at] / c[keep - 1])


def check_sample(logits, u, ids, logp, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows, us = logits.float().cpu().numpy(), u.cpu().numpy()
    ids, logp = ids.cpu().numpy(), None if logp is None else logp.cpu().numpy()
    each = lambda v: v.cpu().numpy() if torch.is_tensor(v) else [v] * len(rows)  # noqa: E731
    t, k, p, q = each(temperature), each(top_k), each(top_p), each(min_p)
    for i, row in enumerate(rows):
        want, lw = plain_sample(row, us[i], float(t[i]), int(k[i]), float(p[i]), float(q[i]))
        assert ids[i] == want, "row %d of %s: id %d, want %d (u=%r, logp %r, want %r)" % (
            i, rows.shape, ids[i], want, us[i], None if logp is None else logp[i], lw)
        if logp is not None:
            assert (logp[i] == lw) if math.isinf(lw) else abs(logp[i] - lw) <= 2.0 ** -24 * abs(lw) + 1e-11, (i, logp[i], lw)


def some_logits(dev, b, v, kind, seed, spread=2.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(b, v, generator=g, device=dev) * (0.3 + spread * torch.rand(b, 1, generator=g, device=dev))
    return x.to(TYPES[kind]), torch.rand(b, generator=g, device=dev), g


SETTINGS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=50), dict(top_k=1000, temperature=1.5), dict(top_p=0.9),
            dict(top_p=0.999, temperature=0.4), dict(top_p=1e-6), dict(min_p=0.05), dict(min_p=1.0),
            dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.02), dict(temperature=50.0, top_k=700, top_p=0.5),
            dict(temperature=0.7, top_k=3000, top_p=0.97, min_p=1e-4), dict(temperature=1e-3, top_p=0.9)]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("b,v", [(1, 1), (3, 2), (5, 63), (2, 64), (4, 257), (300, 100), (33, 1000), (17, 9339), (2, 19724), (3, 50001), (2, 131072)])
def test_sample_sizes_and_settings(dev, b, v, kind):
    from style_transfer_amd import ops
    logits, u, _ = some_logits(dev, b, v, kind, 1000 * b + v)
    for s in SETTINGS:
        ids, logp = ops.sample_logits(logits, u, **s)
        check_sample(logits, u, ids, logp, **s)


def test_sample_many_rows(dev):
    from style_transfer_amd import ops
    logits, u, _ = some_logits(dev, 2100, 777, "bf16", 5)
    for s in (dict(top_k=20, top_p=0.9), dict(top_p=0.8), dict()):
        ids, logp = ops.sample_logits(logits, u, **s)
        check_sample(logits, u, ids, logp, **s)


@pytest.mark.parametrize("b,v", [(100, 131072), (70, 262144), (128, 524288), (127, 16384), (129, 70000)])
def test_sample_parts(dev, b, v):
    """rows in parts of every size, and just too many rows for it (a few of them against the definition)"""
    from style_transfer_amd import ops
    logits, u, _ = some_logits(dev, b, v, "bf16", b)
    for s in (dict(top_p=0.9), dict(top_k=30, temperature=0.7), dict()):
        ids, logp = ops.sample_logits(logits, u, **s)
        pick = [0, 1, b // 2, b - 1]
        check_sample(logits[pick], u[pick], ids[pick], logp[pick], **s)
        assert int(ids.min()) >= 0 and int(ids.max()) < v


def test_sample_many_rows_of_ties(dev):
    """many rows with a top_k: those whose equal logits do not fit into a list, beside rows that do"""
    from style_transfer_amd import ops
    logits, u, g = some_logits(dev, 700, 3001, "f32", 6)
    logits[::3] = torch.randint(0, 3, (3001,), generator=g, device=dev).float()
    logits[5] = -math.inf
    logits[6, 7:] = -math.inf
    for s in (dict(top_k=20, top_p=0.9), dict(top_k=128), dict(top_k=200, min_p=0.01), dict(temperature=0.0), dict(top_k=1)):
        ids, logp = ops.sample_logits(logits, u, **s)
        check_sample(logits, u, ids, logp, **s)


@pytest.mark.parametrize("v", [524288, 262147])
def test_sample_largest_vocabulary(dev, v):
    from style_transfer_amd import ops
    logits, u, _ = some_logits(dev, 2, v, "f32", v)
    for s in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95, temperature=3.0)):
        ids, logp = ops.sample_logits(logits, u, **s)
        check_sample(logits, u, ids, logp, **s)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("v", [100, 9339, 70001])
def test_sample_ties_and_masks(dev, v, kind):
    """rows of one value, of few values, of masked entries (-inf, the type's lowest, NaN), empty rows, infinities, -0 and 0"""
    from style_transfer_amd import ops
    t = TYPES[kind]
    g = torch.Generator(device=dev).manual_seed(v)
    rows = torch.randn(13, v, generator=g, device=dev)
    rows[0] = 0.0
    rows[1] = torch.randint(0, 3, (v,), generator=g, device=dev).float() * 0.5
    rows[2, torch.rand(v, generator=g, device=dev) < 0.7] = -math.inf
    rows[3, torch.rand(v, generator=g, device=dev) < 0.7] = float("nan")
    rows[4] = -math.inf
    rows[5] = float("nan")
    rows[6] = torch.finfo(t).min
    rows[7, 1:] = torch.finfo(t).min
    rows[8, :] = -math.inf
    rows[8, v - 1] = -3.0
    rows[9, torch.rand(v, generator=g, device=dev) < 0.2] = math.inf
    rows[10] = torch.where(torch.rand(v, generator=g, device=dev) < 0.5, -0.0, 0.0)
    rows[11] = torch.finfo(t).max
    rows[11, ::2] = torch.finfo(t).min
    rows[12] = 40 * rows[12]
    logits = rows.to(t)
    u = torch.rand(13, generator=g, device=dev)
    for s in SETTINGS:
        for uu in (u, torch.zeros_like(u), torch.full_like(u, 1 - 2.0 ** -24)):
            ids, logp = ops.sample_logits(logits, uu, **s)
            check_sample(logits, uu, ids, logp, **s)


def test_sample_settings_by_row(dev):
    from style_transfer_amd import ops
    b, v = 96, 5003
    logits, u, g = some_logits(dev, b, v, "f32", 3)
    pick = lambda vals, dt: torch.tensor(vals, dtype=dt, device=dev)[torch.randint(0, len(vals), (b,), generator=g, device=dev)]  # noqa: E731
    s = dict(temperature=pick([0.0, 0.3, 1.0, 2.0], torch.float32), top_k=pick([0, 1, 7, 50, 900, 5003, 100000], torch.int32),
             top_p=pick([0.1, 0.5, 0.9, 1.0], torch.float32), min_p=pick([0.0, 0.01, 0.3], torch.float32))
    ids, logp = ops.sample_logits(logits, u, **s)
    check_sample(logits, u, ids, logp, **s)
    # values that scalars are refused for: as documented for arrays
    odd = dict(temperature=torch.tensor([-1.0, float("nan"), 1.0, 1.0, 1.0, 1.0], device=dev),
               top_k=torch.tensor([0, 0, -5, 0, 0, 0], dtype=torch.int32, device=dev),
               top_p=torch.tensor([1.0, 1.0, float("nan"), 0.0, 2.0, 1.0], device=dev),
               min_p=torch.tensor([0.0, 0.0, float("nan"), 0.0, -1.0, 2.0], device=dev))
    plain = dict(temperature=torch.tensor([0.0, 0.0, 1.0, 1.0, 1.0, 1.0]), top_k=torch.tensor([0, 0, 0, 1, 0, 1]),
                 top_p=torch.ones(6), min_p=torch.zeros(6))
    ids, logp = ops.sample_logits(logits[:6], u[:6], **odd)
    check_sample(logits[:6], u[:6], ids, logp, **plain)


def test_sample_strides_and_alignment(dev):
    from style_transfer_amd import ops
    for kind in sorted(TYPES):
        wide, u, _ = some_logits(dev, 9, 4000, kind, 11)
        for view in (wide[:, 1:3001], wide[:, 3:3002], wide[::2, 5:], wide[:1].expand(9, 4000), wide.t().contiguous().t()[:, :1]):
            ids, logp = ops.sample_logits(view, u[:view.shape[0]].contiguous(), top_k=30, top_p=0.9)
            check_sample(view, u, ids, logp, top_k=30, top_p=0.9)
            ids, logp = ops.sample_logits(view, u[:view.shape[0]].contiguous(), temperature=1.3)
            check_sample(view, u, ids, logp, temperature=1.3)


def test_sample_far_rows(dev):
    """a row that begins past 2^32 bytes"""
    from style_transfer_amd import ops
    v, b = 65536, 20000
    big = torch.zeros(b * v, dtype=torch.bfloat16, device=dev).view(b, v)
    big[b - 1] = torch.randn(v, device=dev).to(torch.bfloat16)
    u = torch.rand(3, device=dev)
    rows = big[[0]].expand(1, v)
    ids, logp = ops.sample_logits(big[b - 3:], u, top_p=0.9)
    check_sample(big[b - 3:], u, ids, logp, top_p=0.9)
    far = big[::b - 1]
    ids, logp = ops.sample_logits(far, u[:2].contiguous(), top_k=10)
    check_sample(far, u[:2], ids, logp, top_k=10)
    del rows


def test_sample_repeats_and_streams(dev):
    """the same answer on every run, on another stream, captured and replayed between eager calls on other inputs"""
    from style_transfer_amd import ops
    sets = [some_logits(dev, 40, 30001, "f32", s)[:2] for s in (1, 2, 3)]
    s = dict(temperature=1.1, top_k=0, top_p=0.95)
    want = [ops.sample_logits(l, u, **s) for l, u in sets]
    for l, u in sets:
        check_sample(l, u, *ops.sample_logits(l, u, **s), **s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.sample_logits(l, u, **s) for l, u in sets]
    torch.cuda.current_stream().wait_stream(side)
    for (a, b), (c, d) in zip(want, got):
        assert torch.equal(a, c) and torch.equal(b, d)
    l0, u0 = sets[0][0].clone(), sets[0][1].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample_logits(l0, u0, **s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_logits(l0, u0, **s)
    for i in (0, 1, 2, 1, 0):
        l0.copy_(sets[i][0]), u0.copy_(sets[i][1])
        graph.replay()
        eager = ops.sample_logits(sets[(i + 1) % 3][0], sets[(i + 1) % 3][1], **s)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])
        assert torch.equal(eager[0], want[(i + 1) % 3][0])


def test_sample_refusals(dev):
    from style_transfer_amd import ops
    logits, u, _ = some_logits(dev, 4, 100, "f32", 1)
    for bad in (dict(temperature=-0.1), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=2.5),
                dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=1.5), dict(top_k=torch.ones(4, device=dev)),
                dict(top_p=torch.ones(3, device=dev)), dict(min_p=torch.ones(4))):
        with pytest.raises(ValueError):
            ops.sample_logits(logits, u, **bad)
    for l, uu in ((logits.double(), u), (logits.t(), u), (logits[0], u), (logits, u[:3]), (logits, u.half()), (logits.cpu(), u),
                  (logits, u.cpu()), (logits[:, :0], u)):
        with pytest.raises(ValueError):
            ops.sample_logits(l, uu)
    ids, logp = ops.sample_logits(logits[:0], u[:0])
    assert ids.shape == (0,) and logp.shape == (0,)
    assert ops.sample_logits(logits, u, want_logp=False)[1] is None


# ---- the product ------------------------------------------------------------------------------------------------------

def codes_of(packed, k):
    c = packed.cpu().numpy()
    return np.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1)[:, :k].astype(np.float64)


def weight_of(codes, scales, zeros, k, group):
    full = lambda a: np.repeat(a.cpu().numpy().astype(np.float64), group, 1)[:, :k]  # noqa: E731
    return (codes_of(codes, k) - (8.0 if zeros is None else full(zeros))) * full(scales)


def some_weight(dev, n, k, group, zeros, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = (0.01 * (0.1 + torch.rand(n, groups, generator=g, device=dev))).half()
    z = torch.randint(0, 16, (n, groups), generator=g, device=dev, dtype=torch.uint8) if zeros else None
    return codes, scales, z, g


def check_product(x, w, bias, y, kind):
    x64, y = x.float().cpu().numpy().astype(np.float64), y.float().cpu().numpy().astype(np.float64)
    b64 = 0.0 if bias is None else bias.cpu().numpy().astype(np.float64)
    want = x64 @ w.T + b64
    A = np.abs(x64) @ np.abs(w).T + np.abs(b64)
    k = x64.shape[1]
    tol = ((k + 64) * 2.0 ** -24 + 2.0 ** -22) * A + 2.0 ** -39 * k * np.abs(x64).max(1, keepdims=True) * np.abs(w).max() + 1e-37
    tol = HALF_STEP[kind] * (np.abs(want) + tol) + tol + (2.0 ** -25 if kind == "f16" else 0.0)   # f16's subnormal step, halved
    far = np.abs(y - want) - tol
    at = np.unravel_index(np.argmax(far), far.shape)
    assert far[at] <= 0, "%s: %r, want %r, may differ by %.3g" % (at, y[at], want[at], tol[at])
    if kind == "f32":
        # and as a whole: K / 32 partial products are added one by one, each addition at random up to 2^-24 of the sum so far, which
        # is of the size sqrt(sum x^2 w^2) where signs are mixed and grows up to |y| where they are not (a row of one sign: 301
        # values of 1.2 make 364, whose own rounding is 2^-25 of 364 and 2^-20 of its sqrt(sum x^2 w^2)): sqrt(K / 32) 2^-24 of
        # both, 2^-20 for K up to 8192
        size = np.linalg.norm(np.sqrt((x64 ** 2) @ (w ** 2).T) + np.abs(b64) + np.abs(want))
        off = np.linalg.norm(y - want)
        assert off <= 2.0 ** -20 * size, "norm of the error %.3g at a size of %.3g" % (off, size)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("m,n,k,group,zeros,bias", [
    (1, 1, 1, 32, False, False), (1, 16, 128, 128, True, True), (2, 17, 33, 32, True, False), (3, 100, 200, 64, False, True),
    (16, 256, 256, 64, True, True), (17, 250, 257, 128, True, True), (31, 64, 1024, 128, False, False), (33, 129, 777, 64, True, True),
    (64, 1000, 96, 32, False, True), (65, 333, 640, 32, True, False), (128, 257, 2049, 128, False, True), (200, 1040, 500, 64, True, True),
    (1, 9339, 256, 32, False, True), (5, 2050, 4096, 128, True, False), (300, 515, 130, 32, False, True), (257, 4100, 1030, 128, True, True)])
def test_gemm_q4(dev, m, n, k, group, zeros, bias, kind):
    from style_transfer_amd import ops
    codes, scales, z, g = some_weight(dev, n, k, group, zeros, m + n + k)
    x = torch.randn(m, k, generator=g, device=dev).to(TYPES[kind])
    b = torch.randn(n, generator=g, device=dev) if bias else None
    q = ops.pack_weight_q4(codes, scales, z, k=k, group=group)
    y = ops.gemm_q4(x, q, b)
    assert y.dtype == x.dtype and y.shape == (m, n)
    check_product(x, weight_of(codes, scales, z, k, group), b, y, kind)
    assert torch.equal(y, ops.gemm_q4(x, q, b))


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("m", [1, 7, 70, 300])
def test_gemm_q4_strides(dev, m, kind):
    """rows of x and y that are apart, that begin off 16 bytes, one row for all; what lies between y's rows stays"""
    from style_transfer_amd import ops
    n, k = 333, 200
    codes, scales, z, g = some_weight(dev, n, k, 64, True, 5)
    q, w = ops.pack_weight_q4(codes, scales, z, group=64), weight_of(codes, scales, z, k, 64)
    wide = torch.randn(m, 408, generator=g, device=dev).to(TYPES[kind])
    for x in (wide[:, :200], wide[:, 8:208], wide[:, 1:201], wide[:1, 4:204].expand(m, 200)):
        check_product(x, w, None, ops.gemm_q4(x, q), kind)
        store = torch.full((m + 1, 350), 7.0, device=dev, dtype=x.dtype)
        assert ops.gemm_q4(x, q, out=store[:m, 3:336]) is not None
        check_product(x, w, None, store[:m, 3:336], kind)
        assert bool((store[:, :3] == 7).all()) and bool((store[:, 336:] == 7).all()) and bool((store[m] == 7).all())


@pytest.mark.parametrize("m", [2, 40, 130])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_gemm_q4_range(dev, m, kind):
    """rows of very small, very large and very unequal values; a row of zeros; infinities and NaN stay in their row"""
    from style_transfer_amd import ops
    n, k = 96, 640
    codes, scales, z, g = some_weight(dev, n, k, 128, False, 9)
    q, w = ops.pack_weight_q4(codes, scales, z), weight_of(codes, scales, z, k, 128)
    x = torch.randn(m, k, generator=g, device=dev)
    for scale in (1e-30, 1e-12, 1e6, 1e30):
        y = (x * scale).to(TYPES[kind])
        check_product(y, w, None, ops.gemm_q4(y, q), kind)
    y = x * torch.exp(8 * torch.randn(m, k, generator=g, device=dev))
    y[1] = 0
    y = y.to(TYPES[kind])
    check_product(y, w, None, ops.gemm_q4(y, q), kind)
    bad = x.clone()
    bad[0, 3], bad[1, 500] = math.inf, float("nan")
    y = ops.gemm_q4(bad.to(TYPES[kind]), q)
    assert not bool(torch.isfinite(y[:2].float()).any()) and bool(torch.isfinite(y[2:].float()).all())
    if m > 2:
        check_product(bad[2:].to(TYPES[kind]), w, None, y[2:], kind)


def test_gemm_q4_far_weights(dev):
    """an image of more than 2^32 codes' bytes is out of reach here, one whose codes pass 2^31 in number is not"""
    from style_transfer_amd import ops
    n, k, m = 131072 + 5, 16384 + 64, 2
    codes, scales, z, g = some_weight(dev, n, k, 128, False, 2)
    x = torch.randn(m, k, generator=g, device=dev).to(torch.bfloat16)
    y = ops.gemm_q4(x, ops.pack_weight_q4(codes, scales, z, k=k))
    for part in (slice(0, 40), slice(n - 40, n)):
        check_product(x, weight_of(codes[part], scales[part], None, k, 128), None, y[:, part], "bf16")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_weight_q4(dev, group, zeros):
    """every weight within half a step of its code's value (a step: the scale), plus the scale's own rounding to f16 times the
    largest code; exact codes against the definition"""
    from style_transfer_amd import ops
    n, k = 37, 301
    g = torch.Generator(device=dev).manual_seed(group)
    W = torch.randn(n, k, generator=g, device=dev) * 0.1
    W[3] = 0
    W[4, :group] = 0.7
    W[5] = W[5].abs() + 1.0
    codes, scales, z = ops.quantize_weight_q4(W, group, zeros)
    assert (z is not None) == zeros
    w, want = weight_of(codes, scales, z, k, group), W.cpu().numpy().astype(np.float64)
    s = np.repeat(scales.cpu().numpy().astype(np.float64), group, 1)[:, :k]
    assert (np.abs(w - want) <= 0.5 * s * (1 + 2.0 ** -20) + 15 * s * 2.0 ** -11 + (0.5 * s if zeros else 0)).all()
    assert (w[3] == 0).all()
    if not zeros:
        a = np.abs(want)
        for i in range(0, k, group):
            step = (a[:, i:i + group].max(1).astype(np.float32) / np.float32(7)).astype(np.float16)
            assert np.array_equal(step, scales[:, i // group].cpu().numpy())
    y = ops.gemm_q4(W[:9].contiguous(), ops.pack_weight_q4(codes, scales, z, k=k, group=group))
    check_product(W[:9], w, None, y, "f32")


@pytest.mark.parametrize("m", [1, 40])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_weight_q4_not_finite(dev, zeros, m):
    """a weight that 4 bits and an f16 scale cannot hold is seen in the product, in its row alone"""
    from style_transfer_amd import ops
    g = torch.Generator(device=dev).manual_seed(5)
    W = torch.randn(12, 96, generator=g, device=dev)
    W[1, 40], W[4, 0], W[5, 95], W[7, 33], W[9, 64] = float("nan"), float("inf"), -float("inf"), 2.0e6, -3.0e38
    W[9, 65] = 3.0e38                      # the range itself is beyond f32
    codes, scales, z = ops.quantize_weight_q4(W, 32, zeros)
    x = torch.randn(m, 96, generator=g, device=dev)
    y = ops.gemm_q4(x, ops.pack_weight_q4(codes, scales, z, group=32))
    bad = [1, 4, 5, 7, 9]
    good = [i for i in range(12) if i not in bad]
    assert not torch.isfinite(y[:, bad]).any()
    check_product(x, weight_of(codes[good], scales[good], None if z is None else z[good], 96, 32), None, y[:, good], "f32")


def test_gemm_q4_graph_and_stream(dev):
    from style_transfer_amd import ops
    codes, scales, z, g = some_weight(dev, 1000, 512, 64, True, 4)
    q = ops.pack_weight_q4(codes, scales, z, group=64)
    for m in (3, 150):
        xs = [torch.randn(m, 512, generator=g, device=dev) for _ in range(3)]
        want = [ops.gemm_q4(x, q) for x in xs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [ops.gemm_q4(x, q) for x in xs]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        x0 = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.gemm_q4(x0, q)
        for i in (0, 2, 1, 0):
            x0.copy_(xs[i])
            graph.replay()
            again = ops.gemm_q4(xs[(i + 1) % 3], q)
            torch.cuda.synchronize()
            assert torch.equal(y, want[i]) and torch.equal(again, want[(i + 1) % 3])


def test_q4_refusals(dev):
    from style_transfer_amd import ops
    codes, scales, z, g = some_weight(dev, 40, 128, 64, True, 1)
    q = ops.pack_weight_q4(codes, scales, z, group=64)
    x = torch.randn(4, 128, device=dev)
    for args, kw in (((codes, scales), dict(group=48)), ((codes, scales), dict(group=128)), ((codes, scales.float()), dict(group=64)),
                     ((codes, scales, z[:, :1]), dict(group=64)), ((codes.cpu(), scales), dict(group=64)), ((codes, scales), dict(group=64, k=200)),
                     ((codes.t(), scales), dict(group=64)), ((codes, scales, z.cpu()), dict(group=64))):
        with pytest.raises(ValueError):
            ops.pack_weight_q4(*args, **kw)
    for a, kw in ((x[:, :100], {}), (x.double(), {}), (x.t(), {}), (x[0], {}), (x.cpu(), {}), (x, dict(bias=torch.zeros(39, device=dev))),
                  (x, dict(bias=torch.zeros(40, device=dev).half())), (x, dict(out=torch.empty(4, 41, device=dev))),
                  (x, dict(out=torch.empty(4, 40, device=dev).half())), (x, dict(out=torch.empty(40, 4, device=dev).t()))):
        with pytest.raises(ValueError):
            ops.gemm_q4(a, q, **kw)
    for W, kw in ((x.half(), {}), (x.t(), {}), (x, dict(group=16)), (x[:0], {})):
        with pytest.raises(ValueError):
            ops.quantize_weight_q4(W, **kw)
    assert ops.gemm_q4(x[:0], q).shape == (0, 40)


def test_gemm_q4_out_and_x_in_one_buffer(dev):
    from style_transfer_amd import ops
    codes, scales, z, g = some_weight(dev, 128, 128, 64, True, 2)
    q = ops.pack_weight_q4(codes, scales, z, group=64)
    buf = torch.randn(40, 300, generator=g, device=dev)
    want = ops.gemm_q4(buf[:, :128], q)
    for a, b in ((buf[:, :128], buf[:, :128]), (buf[:, :128], buf[:, 100:228]), (buf[1:, :128], buf[:39, :128])):
        with pytest.raises(ValueError, match="shares"):
            ops.gemm_q4(a, q, out=b)
    ops.gemm_q4(buf[:, :128], q, out=buf[:, 130:258])
    assert torch.equal(buf[:, 130:258], want)


# ---- in a row ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 64, 200])
def test_head_and_draw(dev, rows):
    """quantised head -> logits -> tokens, as a decode step uses them: the draw of the very logits that the product gave"""
    from style_transfer_amd import ops
    V, g = 9339, torch.Generator(device=dev).manual_seed(rows)
    W, b = torch.randn(V, 256, generator=g, device=dev) * 0.2, torch.randn(V, generator=g, device=dev) * 0.1
    codes, scales, z = ops.quantize_weight_q4(W, 64)
    q = ops.pack_weight_q4(codes, scales, z, group=64)
    h, u = torch.randn(rows, 256, generator=g, device=dev), torch.rand(rows, generator=g, device=dev)
    logits = ops.gemm_q4(h, q, b)
    check_product(h, weight_of(codes, scales, z, 256, 64), b, logits, "f32")
    s = dict(temperature=0.9, top_k=60, top_p=0.95)
    ids, logp = ops.sample_logits(logits, u, **s)
    check_sample(logits, u, ids, logp, **s)
    ids0, _ = ops.sample_logits(logits, u, temperature=0.0)
    assert torch.equal(ids0.long(), logits.argmax(1))


# ---- the decoder's loop with draws --------------------------------------------------------------------------------------

@pytest.fixture(scope="module", params=["f16x3", "f32"])
def ae(request, ae_sd_torch, dev):
    from style_transfer_amd.weights import AEWeights
    return AEWeights(ae_sd_torch, dev, gemm_format=request.param)


@pytest.fixture(scope="module")
def latents(dev):
    from conftest import gold
    z = gold("attack_notnll.npz")["latent"].reshape(-1, 256).astype(np.float32)
    return torch.from_numpy(np.ascontiguousarray(z[:: max(1, len(z) // 60)][:60])).to(dev)


def lengths_of(ids):
    """tokens of each row up to its first EOS / PAD, that one included"""
    return [next((i + 1 for i, x in enumerate(r) if x in (0, 3)), len(r)) for r in ids]


def test_sample_decode_greedy(dev, ae, latents):
    """temperature 0 (for all, and for every other sentence between sampled ones): greedy_decode's tokens, log-probability 0.
    (Where the two best logits are closer than the products' rounding, 1e-3, the two may part.)"""
    from style_transfer_amd import ops
    B = latents.shape[0]
    g = torch.Generator(device=dev).manual_seed(1)
    u = torch.rand(B, 59, generator=g, device=dev)
    ids, gap, _ = ops.greedy_decode(ae, latents, want_gap=True)
    ids, gap = ids.cpu().numpy(), gap.cpu().numpy()
    alone, logp, steps = ops.sample_decode(ae, latents, u, temperature=0.0)
    assert bool((logp == 0).all()) and steps > 0
    t = torch.where(torch.arange(B, device=dev) % 2 == 0, 0.0, 1.0)
    mixed, _, _ = ops.sample_decode(ae, latents, u, temperature=t)
    same = 0
    for s, n in enumerate(lengths_of(ids)):
        if gap[s, :n].min() <= 1e-3:
            continue
        same += 1
        assert np.array_equal(alone[s, :n].cpu().numpy(), ids[s, :n]), s
        assert bool((alone[s, n:] == 0).all())
        if s % 2 == 0:
            assert np.array_equal(mixed[s, :n].cpu().numpy(), ids[s, :n]), s
    assert same > B // 2


@pytest.mark.parametrize("head_bits", [0, 4])
def test_sample_decode_draws(dev, ae, ae_sd, latents, head_bits):
    """every drawn token against the CPU oracle's logits for the tokens before it (with the 4-bit head: of the weights that the codes
    stand for): its log-probability within 1e-2, and u between the masses before and behind it within 1e-2 (logits are good to 2e-4
    of the largest, about 30, which moves a share by 2 x 6e-3 of itself at most)"""
    import st_oracle as O
    from style_transfer_amd import ops
    sd, head = dict(ae_sd), None
    if head_bits:
        W = torch.from_numpy(np.ascontiguousarray(ae_sd["generator.proj.weight"])).to(dev)
        codes, scales, z = ops.quantize_weight_q4(W, 64, True)
        sd["generator.proj.weight"] = weight_of(codes, scales, z, 256, 64).astype(np.float32)
        head = ae.quantized_generator(64, True)
    z = latents[:20]
    g = torch.Generator(device=dev).manual_seed(7 + head_bits)
    u = torch.rand(20, 59, generator=g, device=dev)
    pe = O.positional_encoding(60)
    for s in (dict(temperature=1.0), dict(temperature=1.3, top_k=8), dict(temperature=0.9, top_p=0.8, min_p=0.01)):
        ids, logp, _ = ops.sample_decode(ae, z, u, head=head, **s)
        again, logp2, _ = ops.sample_decode(ae, z, u, head=head, **s)
        assert torch.equal(ids, again) and torch.equal(logp, logp2)
        few, _, _ = ops.sample_decode(ae, z[3:5].contiguous(), u[3:5].contiguous(), head=head, **s)
        assert torch.equal(few, ids[3:5])                       # a sentence's draws are its own, whoever is decoded with it
        ids, logp, un = ids.cpu().numpy(), logp.cpu().numpy(), u.cpu().numpy()
        ys = np.concatenate([np.full((20, 1), 2), ids[:, :-1]], 1).astype(np.int64)
        logits = O.linear(O.decode_full(sd, z.cpu().numpy(), ys, pe), sd, "generator.proj").astype(np.float64)
        for b, n in enumerate(lengths_of(ids)):
            assert (ids[b, n:] == 0).all() and (logp[b, n:] == 0).all()
            for t in range(n):
                row, k = logits[b, t], ids[b, t]
                order = np.argsort(-row, kind="stable")
                if s.get("top_k"):
                    order = order[:s["top_k"]]
                w = np.exp((row[order] - row[order[0]]) / s["temperature"])
                c = np.cumsum(w)
                keep = int(np.searchsorted(np.concatenate(([0.0], c))[:-1], s.get("top_p", 1.0) * c[-1] * (1 + 1e-12))) if "top_p" in s else len(w)
                keep = max(1, min(keep, int((w >= s.get("min_p", 0.0)).sum())))
                at = int(np.nonzero(order == k)[0][0]) if k in order[:min(len(order), keep + 2)] else -1
                assert at >= 0, "sentence %d token %d: %d is not among the kept ones" % (b, t, k)
                # an entry at the border may be kept by one side alone: shares go by the set that has the token
                S = c[max(keep - 1, at)]
                assert abs(logp[b, t] - math.log(w[at] / S)) < 1e-2 + 2 * w[keep - 1] / S, (b, t)
                slack = 1e-2 + 2 * w[keep - 1] / S * (keep < len(w))
                assert (c[at] - w[at]) / S - slack <= un[b, t] <= c[at] / S + slack, (b, t, un[b, t], c[at] / S)


def test_sample_decode_large_vocabulary_and_batches(dev, ae_sd_torch):
    """more live rows than logits are held at a time, steps that end rows, and the parts of long rows: a sentence draws the same tokens
    in any batch"""
    from conftest import GOLD
    import os
    from style_transfer_amd import ops, weights as W
    sd = W.expand_ae_state_dict(W.load_state_dict_file(os.path.join(GOLD, "surrogate_ae_amazon.safetensors")))
    ae = W.AEWeights(sd, dev, l0_table=False)
    g = torch.Generator(device=dev).manual_seed(3)
    from conftest import gold
    z = torch.from_numpy(gold("attack_amazon.npz")["latent"].reshape(-1, 256).astype(np.float32)).to(dev)
    z = z[torch.randint(0, z.shape[0], (3700,), generator=g, device=dev)].contiguous()
    u = torch.rand(3700, 59, generator=g, device=dev)
    s = dict(temperature=0.8, top_p=0.9)
    head = ae.quantized_generator()
    ids, logp, _ = ops.sample_decode(ae, z, u, head=head, **s)
    assert bool(torch.isfinite(logp).all()) and bool((logp <= 0).all()) and int(ids.min()) >= 0 and int(ids.max()) < ae.vocab
    pick = torch.tensor([0, 1, 1700, 3390, 3699], device=dev)
    few, lf, _ = ops.sample_decode(ae, z[pick].contiguous(), u[pick].contiguous(), head=head, **s)
    assert torch.equal(few, ids[pick]) and bool(((lf - logp[pick]).abs() < 1e-3).all())


def test_sample_decode_refusals(dev, ae, latents):
    from style_transfer_amd import ops
    z, u = latents[:4].contiguous(), torch.rand(4, 59, device=dev)
    head = ae.quantized_generator()
    wrong = ops.pack_weight_q4(*ops.quantize_weight_q4(torch.randn(100, 256, device=dev)))
    for a, b, kw in ((z.half(), u, {}), (z[:, :100], u, {}), (z, u[:, :58], {}), (z, u[:3], {}), (z, u.double(), {}), (z.cpu(), u, {}),
                     (z, u, dict(head=wrong)), (z, u, dict(head=head.image)), (z, u, dict(top_p=0.0)), (z, u, dict(temperature=-1.0)),
                     (z, u, dict(top_k=torch.ones(3, dtype=torch.int32, device=dev)))):
        with pytest.raises(ValueError):
            ops.sample_decode(ae, a, b, **kw)
    ids, logp, steps = ops.sample_decode(ae, z[:0], u[:0])
    assert ids.shape == (0, 59) and steps == 0


# ---- more rows, settings and inputs that the documentation allows -------------------------------------------------------

@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("b", [511, 512, 513])
@pytest.mark.parametrize("v", [257, 300, 777, 1000, 1024, 1025, 2600])
def test_sample_many_short_rows_masked(dev, b, v, kind):
    """many rows with a top_k, on both sides of every size at which another kernel takes them: rows with none, one, a few, top_k - 1,
    top_k and all of their entries left, the entries side by side or spread out, and rows of ties; one setting for all and arrays"""
    from style_transfer_amd import ops
    logits, u, g = some_logits(dev, b, v, kind, b + v)
    k = max(2, min(50, v // 12))
    live = torch.tensor([0, 1, 3, k - 1, k, v], device=dev)[torch.arange(b, device=dev) % 6]
    place = torch.arange(v, device=dev).repeat(b, 1)
    place[b // 2:] = torch.rand(b - b // 2, v, generator=g, device=dev).argsort(1)
    masked = torch.tensor([-math.inf, float("nan")], device=dev, dtype=logits.dtype)[torch.arange(b, device=dev) % 2][:, None]
    logits = torch.where(place < live[:, None], logits, masked)
    logits[5::12] = torch.randint(0, 3, (v,), generator=g, device=dev).to(logits.dtype)
    ks = torch.tensor([k, 0, 1, k + 7, v], dtype=torch.int32, device=dev)[torch.randint(0, 5, (b,), generator=g, device=dev)]
    for s in (dict(top_k=k, top_p=0.9), dict(top_k=k, min_p=0.01, temperature=1.4), dict(top_k=ks, temperature=0.8), dict(top_k=1)):
        ids, logp = ops.sample_logits(logits, u, **s)
        assert int(ids.min()) == -1
        check_sample(logits, u, ids, logp, **s)


def rows_of_the_whole_range(dev, v, kind, seed):
    """rows whose largest and smallest logits are farther apart than f32's largest number (f16's own range is 131008 wide)"""
    g = torch.Generator(device=dev).manual_seed(seed)
    most = torch.finfo(TYPES[kind]).max
    at = torch.rand(12, v, generator=g, device=dev)
    rows = at * 2 * (most / 2) - most / 2
    rows[0:4] = torch.where(at[0:4] < 0.5, 0.88 * most, -0.88 * most)
    rows[4:8] = torch.where(at[4:8] < 0.5, most, -most)
    rows[8:10] *= 1.99
    rows[10, ::3] = -math.inf
    rows[11, ::3] = math.inf
    u = torch.rand(12, generator=g, device=dev)
    u[::2] = 1 - 2.0 ** -24               # among the last entries, far from the top
    return rows.to(TYPES[kind]), u


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("v", [300, 3000, 9339, 40000])
def test_sample_whole_range_of_logits(dev, v, kind):
    """temperatures from which logits at both ends of the type share the mass"""
    from style_transfer_amd import ops
    logits, u = rows_of_the_whole_range(dev, v, kind, v)
    for t in (3e4, 1.05e37, 1.07e37, 3e37, 1e38):
        for s in (dict(), dict(top_k=700), dict(top_p=0.9), dict(top_k=20), dict(min_p=0.3)):
            ids, logp = ops.sample_logits(logits, u, temperature=t, **s)
            check_sample(logits, u, ids, logp, temperature=t, **s)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("v", [300, 3000, 40000])
def test_sample_largest_temperatures(dev, v, kind):
    """f32's largest temperature, and an infinite one in an array: every finite logit has the same weight"""
    from style_transfer_amd import ops
    logits, u = rows_of_the_whole_range(dev, v, kind, v + 1)
    logits = logits[:11]
    u = u[:11].contiguous()
    for t in (torch.finfo(torch.float32).max, torch.full((11,), torch.finfo(torch.float32).max, device=dev), torch.full((11,), math.inf, device=dev)):
        for s in (dict(), dict(top_k=700), dict(top_p=0.9), dict(top_k=20), dict(min_p=0.3)):
            ids, logp = ops.sample_logits(logits, u, temperature=t, **s)
            check_sample(logits, u, ids, logp, temperature=t, **s)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k,outlier", [(47, 64, 90, 0), (47, 64, 90, 89), (47, 100, 700, 3), (47, 100, 1500, 1499), (256, 4100, 6200, 0), (256, 4100, 6200, 6199)])
def test_gemm_q4_small_values_beside_an_outlier(dev, m, n, k, outlier, kind):
    """one value of a row is far larger than the others and has weight 0 (its code is the zero code): what is left is the others'
    product, each with an error of 2^-39 of the outlier at most, f32 ones of 2^-22 of themselves if that is more, beside the f32
    sums' own (all x and w positive, so that errors of one direction add up, and mixed signs).
    (f32: hi takes 11 bits of a value of the power 2^e, cut off; less than 2^(e - 10) is left, of which 11 bits are kept to the
    nearest: half a step is 2^(e - 11 - 10 - 1) = 2^(e - 22).  Subnormals: half of 2^-24 where the outlier is 2^14.)"""
    from style_transfer_amd import ops
    g = torch.Generator(device=dev).manual_seed(m + k + outlier)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = (0.01 * (0.1 + torch.rand(n, -(-k // 64), generator=g, device=dev))).half()
    for signs in (False, True):
        c = codes if signs else codes | 0x88
        at, keep = outlier // 2, 0xf0 if outlier % 2 == 0 else 0x0f
        c = c.clone()
        c[:, at] = (c[:, at] & keep) | (0x88 & ~keep)
        far = 2.0 ** -(torch.arange(m, device=dev) % 47).float()[:, None]
        x = far * (1 + torch.rand(m, k, generator=g, device=dev))
        if signs:
            x = torch.where(torch.rand(m, k, generator=g, device=dev) < 0.5, x, -x)
        x[:, outlier] = 1.0
        x = x.to(TYPES[kind])
        y = ops.gemm_q4(x, ops.pack_weight_q4(c, scales, group=64), None).float().cpu().numpy().astype(np.float64)
        w, x64 = weight_of(c, scales, None, k, 64), x.float().cpu().numpy().astype(np.float64)
        assert (w[:, outlier] == 0).all()
        want, a = x64 @ w.T, np.abs(w)
        value = np.maximum((2.0 ** -22 if kind == "f32" else 0.0) * np.abs(x64), 2.0 ** -39 * np.abs(x64).max(1, keepdims=True))
        tol = value @ a.T + (k + 64) * 2.0 ** -24 * (np.abs(x64) @ a.T)
        tol += HALF_STEP[kind] * (np.abs(want) + tol)
        over = np.abs(y - want) - tol
        i = np.unravel_index(np.argmax(over), over.shape)
        assert over[i] <= 0, "%s: %r, want %r, may differ by %.3g" % (i, y[i], want[i], tol[i])


def test_quantized_generator_of_weights_that_train_on(dev, ae_sd_torch):
    """the 4-bit head is that of the weights that were packed, whatever the caller does with its tensors afterwards"""
    from style_transfer_amd.weights import AEWeights
    sd = {k: v.clone() for k, v in ae_sd_torch.items()}
    want = AEWeights(ae_sd_torch, dev, l0_table=False).quantized_generator(32, True).image
    ae = AEWeights(sd, dev, l0_table=False)
    sd["generator.proj.weight"].mul_(3.0).add_(1.0)
    assert torch.equal(ae.quantized_generator(32, True).image, want)


def test_gemm_q4_refuses_to_lose_a_gradient(dev):
    from style_transfer_amd import ops
    codes, scales, z, g = some_weight(dev, 40, 128, 64, True, 1)
    q = ops.pack_weight_q4(codes, scales, z, group=64)
    x, bias = torch.randn(4, 128, generator=g, device=dev), torch.randn(40, generator=g, device=dev)
    want = ops.gemm_q4(x, q, bias)
    leaf, row = x.clone().requires_grad_(), bias.clone().requires_grad_()
    for a, b in ((leaf, None), (leaf * 1.0, bias), (x, row)):
        with pytest.raises(ValueError, match="gradient"):
            ops.gemm_q4(a, q, b)
    with torch.no_grad():
        assert torch.equal(ops.gemm_q4(leaf, q, row), want)
    with torch.inference_mode():
        assert torch.equal(ops.gemm_q4(leaf, q, row), want)
    assert torch.equal(ops.gemm_q4(leaf.detach(), q, bias), want)


def test_sample_decode_refuses_weights_elsewhere(dev, ae, latents):
    import copy
    from style_transfer_amd import ops
    assert ae.where == latents.device
    other = copy.copy(ae)
    other.where = torch.device("cuda", 1)
    with pytest.raises(ValueError, match="weights are on"):
        ops.sample_decode(other, latents[:2].contiguous(), torch.rand(2, 59, device=dev))


@pytest.mark.parametrize("head_bits", [0, 4])
def test_sample_decode_range_error_names_its_entry_point(dev, ae_sd_torch, head_bits):
    from style_transfer_amd import _lib, ops
    from style_transfer_amd.weights import AEWeights
    sd = {k: v.clone() for k, v in ae_sd_torch.items()}
    sd["decoder.layers.1.feed_forward.w_1.weight"] *= 3e4
    ae = AEWeights(sd, dev, l0_table=False)
    latent, u = torch.rand(48, 256, device=dev) * 8, torch.rand(48, 59, device=dev)
    with pytest.raises(_lib.StError, match="f16 range") as e:
        ops.sample_decode(ae, latent, u, head=ae.quantized_generator() if head_bits else None)
    assert "st_decode_greedy" not in str(e.value)
    with pytest.raises(_lib.StError, match="st_decode_greedy: an activation"):
        ops.greedy_decode(ae, latent)


def test_sizes_beyond_32_bits_are_refused(dev):
    """the C entry points take 32-bit sizes: 2^32 + 3 rows are not 3 rows"""
    from style_transfer_amd import ops
    far, u = (1 << 32) + 3, torch.rand(3, device=dev)
    with pytest.raises(ValueError, match="32 bits"):
        ops.sample_logits(torch.zeros(1, 1, device=dev).expand(far, 1), u)
    q = ops.pack_weight_q4(*ops.quantize_weight_q4(torch.ones(4, 8, device=dev), 32), k=8, group=32)
    for m in ((1 << 20), far):
        with pytest.raises(ValueError, match="at most"):
            ops.gemm_q4(torch.zeros(1, 8, device=dev).expand(m, 8), q)
    with pytest.raises(ValueError, match="at most"):
        ops.quantize_weight_q4(torch.empty(far, 1, device=dev), 32)
    with pytest.raises(ValueError, match="at most"):
        ops.quantize_weight_q4(torch.empty(1, (1 << 24) + 1, device=dev), 32)
    with pytest.raises(ValueError, match="at most"):
        ops.pack_weight_q4(torch.empty(far, 1, device=dev, dtype=torch.uint8), torch.empty(1, 1, device=dev, dtype=torch.float16).expand(far, 1), group=32)


def test_quantize_weight_q4_of_2_32_values(dev):
    """more groups than a launch has waves for: rows from all over against the same rows by themselves"""
    from style_transfer_amd import ops
    n, k = 262144 + 3, 16384
    W = torch.empty(n, k, device=dev)
    for i in range(0, n, 32768):
        W[i:i + 32768].normal_(0, 0.1, generator=torch.Generator(device=dev).manual_seed(i))
    codes, scales, zeros = ops.quantize_weight_q4(W, 32, True)
    for part in (slice(0, 50), slice(n // 4 - 25, n // 4 + 25), slice(n // 2 - 25, n // 2 + 25), slice(n - 50, n)):
        c, s, z = ops.quantize_weight_q4(W[part].clone(), 32, True)
        assert torch.equal(c, codes[part]) and torch.equal(s, scales[part]) and torch.equal(z, zeros[part])


def test_pack_weight_q4_of_2_35_codes(dev):
    """an image of 2^34 bytes and more: its first, middle and last rows in a product"""
    from style_transfer_amd import ops
    n, k = (1 << 20) + 5, 32768
    g = torch.Generator(device=dev).manual_seed(3)
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device=dev)
    for i in range(0, n, 131072):
        codes[i:i + 131072] = torch.randint(0, 256, codes[i:i + 131072].shape, generator=g, device=dev, dtype=torch.uint8)
    scales = (0.01 * (0.1 + torch.rand(n, k // 128, generator=g, device=dev))).half()
    x = torch.randn(2, k, generator=g, device=dev).half()
    y = ops.gemm_q4(x, ops.pack_weight_q4(codes, scales))
    for part in (slice(0, 40), slice(n // 2 - 20, n // 2 + 20), slice(n - 40, n)):
        check_product(x, weight_of(codes[part], scales[part], None, k, 128), None, y[:, part], "f16")


def test_gemm_q4_out_and_bias_in_one_buffer(dev):
    from style_transfer_amd import ops
    codes, scales, z, g = some_weight(dev, 128, 128, 64, True, 2)
    q = ops.pack_weight_q4(codes, scales, z, group=64)
    x, buf = torch.randn(40, 128, generator=g, device=dev), torch.randn(40, 300, generator=g, device=dev)
    want = ops.gemm_q4(x, q, buf[3, 150:278].clone())
    for bias in (buf[3, :128], buf[0, 100:228], buf[39, 127:255]):
        with pytest.raises(ValueError, match="shares values with bias"):
            ops.gemm_q4(x, q, bias, out=buf[:, :128])
    with pytest.raises(ValueError, match="shares values with bias"):
        ops.gemm_q4(x[:1].bfloat16(), q, buf[3, :128], out=buf.view(torch.bfloat16)[3:4, 254:382])
    ops.gemm_q4(x, q, buf[3, 150:278], out=buf[:, :128])       # beside the columns that are written
    assert torch.equal(buf[:, :128], want)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_weight_q4_codes(dev, group, zeros):
    """scales, zero codes and codes equal to the definition's: the scale in f32 and then f16, a code the nearest whole number of
    scales above the zero code, 0 to 15, ties to even (f32 quotients, as the definition has them); odd columns and a short last group"""
    from style_transfer_amd import ops
    n, k = 29, 301
    g = torch.Generator(device=dev).manual_seed(group + zeros)
    W = torch.randn(n, k, generator=g, device=dev) * torch.exp(3 * torch.randn(n, 1, generator=g, device=dev))
    W[3], W[4], W[5], W[6] = 0, 0.7, W[5].abs() + 1.0, -W[6].abs() - 1.0
    W[7], W[8] = W[7] * 1e-7, W[8] * 1e-12             # scales that are f16 subnormals, or 0
    W[9] = torch.randint(-7, 8, (k,), generator=g, device=dev).float() * 0.5   # ties and exact codes
    codes, scales, z = ops.quantize_weight_q4(W, group, zeros)
    w, got = W.cpu().numpy(), codes_of(codes, k)
    f = np.float32
    for i in range(n):
        for j in range(0, k, group):
            v = w[i, j:j + group]
            hi, lo = f(max(v.max(), 0)), f(min(v.min(), 0))
            step = (f(hi - lo) / f(15) if zeros else max(hi, -lo) / f(7)).astype(np.float16)
            s, at = f(step), j // group
            assert scales[i, at].cpu().numpy() == step, (i, j)
            zero = 8
            if zeros:
                zero = int(np.clip(np.rint(-lo / s), 0, 15)) if s > 0 else 0
                assert int(z[i, at]) == zero, (i, j)
            want = np.clip(np.clip(np.rint(v / s), -16, 16) + zero, 0, 15) if s > 0 else np.full(len(v), zero)
            assert np.array_equal(got[i, j:j + group], want), (i, j)


def test_sample_workspace_in_graphs(dev):
    """two graphs captured with one DecodeWorkspace, which a larger call replaces before they are replayed, side by side"""
    from style_transfer_amd import ops
    ws, s = ops.DecodeWorkspace(dev), dict(top_p=0.95)
    sets = [some_logits(dev, 40, 30001, "f32", i)[:2] for i in (1, 2)]
    want = [ops.sample_logits(l, u, ws=ws, **s) for l, u in sets]
    first = ws.buf.data_ptr(), ws.buf.numel()
    graphs, outs = [], []
    for l, u in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.sample_logits(l, u, ws=ws, **s))
    big = some_logits(dev, 2, 400000, "bf16", 3)[:2]
    assert ws.buf.data_ptr() == first[0]
    ws.get(first[1] + (8 << 20))
    other = torch.full((first[1],), 7, dtype=torch.uint8, device=dev)      # where the first one was
    side = torch.cuda.Stream()
    for _ in range(5):
        for o in outs:
            o[0].fill_(-9)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        ids, logp = ops.sample_logits(*big, ws=ws, **s)
        torch.cuda.synchronize()
        check_sample(*big, ids, logp, **s)
        for o, w in zip(outs, want):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
    assert bool((other == 7).all())


def test_sample_workspace_replaced_while_another_stream_uses_it(dev):
    from style_transfer_amd import ops
    logits, u, _ = some_logits(dev, 40, 30001, "f32", 1)
    want = ops.sample_logits(logits, u, top_p=0.95)
    ws = ops.DecodeWorkspace(dev)
    at, n = ws.get(ops.lib().st_sample_workspace_bytes(40, 30001)).data_ptr(), ws.buf.numel()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                      # about a tenth of a second before the draw starts
        got = ops.sample_logits(logits, u, top_p=0.95, ws=ws)
    ws.get(n + (8 << 20))
    other = torch.empty(n, dtype=torch.uint8, device=dev)
    assert not side.query() and other.data_ptr() != at      # the old buffer still belongs to the draw
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
