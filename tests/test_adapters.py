"""Low-rank adapters of many requests beside a shared projection (ops.adapter_gemm / adapter_gemm_backward): the HIP kernels against
the formulas in 64 bits, element by element, under bounds that count the kernels' own roundings.

With u = eps / 2 of the operand type: a 16-bit result rounds the low-rank values once and the result once, so
|error| <= u (sum_j |low_j up_j| + |out|); where the low-rank values are kept as planes they are off by u^2 (fp16: two planes) or
u^3 (bf16: three), and by 2^-25 absolutely where an fp16 remainder is below its normal range (2^-36 in the gradient's t, whose
remainder plane is scaled by 2^11).  Sums are fp32: n terms are off by at most n 2^-24 of the sum of their
magnitudes, taken here as sqrt(n) + 8 steps, which a random walk of that many roundings does not pass (each is at most half a
step of the running sum)."""
import ctypes
import math

import pytest
import torch

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch.device("cuda:0")


def rnd(shape, dev, dtype, seed, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dev).to(dtype)


def acc(n):
    return (math.sqrt(n) + 8) * 2.0 ** -24


def reference(a, w, down, up, who, scale, bias, residual, out_f32, dout=None):
    """(values, bounds), dicts of fp64 tensors: out, low and, with dout, da, ddown, dup — from the formulas.  who: adapter of each row."""
    dt = a.dtype
    u = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    M, K = a.shape
    S, r, _ = down.shape
    N = w.shape[0]
    A, W, D, U = (x.double() for x in (a, w, down, up))
    base = A @ W.t()
    absbase = A.abs() @ W.t().abs()
    low, lowabs = (torch.zeros((M, r), dtype=torch.float64, device=a.device) for _ in range(2))
    add, addabs, addlow = (torch.zeros((M, N), dtype=torch.float64, device=a.device) for _ in range(3))
    p = u * u if dt == torch.float16 else u ** 3
    res = {}
    if dout is not None:
        dY = dout.double()
        t, tabs = torch.zeros_like(low), torch.zeros_like(low)
        da, daabs, dalow = (torch.zeros((M, K), dtype=torch.float64, device=a.device) for _ in range(3))
        ddown, eddown = (torch.zeros((S, r, K), dtype=torch.float64, device=a.device) for _ in range(2))
        dup, edup = (torch.zeros((S, N, r), dtype=torch.float64, device=a.device) for _ in range(2))
    for i in range(S):
        at = (who == i).nonzero()[:, 0]
        if at.numel() == 0:
            continue
        s = float(scale[i]) if scale is not None else 1.0
        low[at] = s * A[at] @ D[i].t()
        lowabs[at] = s * A[at].abs() @ D[i].t().abs()
        add[at] = low[at] @ U[i].t()
        addabs[at] = low[at].abs() @ U[i].t().abs()
        elow = acc(K) * lowabs[at] + (p * low[at].abs() + tiny if out_f32 else u * low[at].abs() + tiny)
        addlow[at] = elow @ U[i].t().abs()
        if dout is None:
            continue
        t[at] = s * dY[at] @ U[i]
        tabs[at] = s * dY[at].abs() @ U[i].abs()
        da[at] = t[at] @ D[i]
        dalow[at] = (u * t[at].abs() + tiny + acc(N) * tabs[at]) @ D[i].abs()
        daabs[at] = t[at].abs() @ D[i].abs()
        e_t = acc(N) * tabs[at] + p * t[at].abs() + tiny * 2.0 ** -11
        e_u = acc(K) * lowabs[at] + p * low[at].abs() + tiny
        n = acc(at.numel())
        ddown[i] = t[at].t() @ A[at]
        eddown[i] = (e_t + n * t[at].abs()).t() @ A[at].abs()
        dup[i] = dY[at].t() @ low[at]
        edup[i] = dY[at].abs().t() @ (e_u + n * low[at].abs())
    out = base + add
    size = absbase + addabs
    for x in (bias, residual):
        if x is not None:
            out = out + x.double()
            size = size + x.double().abs()
    err = addlow + acc(K + r) * size
    res_b = dict(out=err + (2.0 ** -24 * out.abs() if out_f32 else u * (out.abs() + err) + tiny))
    res = dict(out=out)
    if dout is not None:
        da_all = dY @ W + da
        err = dalow + acc(N + r) * (dY.abs() @ W.abs() + daabs)
        res.update(da=da_all, ddown=ddown, dup=dup)
        res_b.update(da=err + u * (da_all.abs() + err) + tiny, ddown=eddown * 1.01 + 1e-30, dup=edup * 1.01 + 1e-30)
    return res, res_b


def within(name, got, val, bnd):
    assert got.shape == val.shape, name
    bad = ~((got.double() - val).abs() <= bnd)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()}, worst error / bound " \
                          f"{float(((got.double() - val).abs() / bnd.clamp_min(1e-300))[bad].max()):.3g}, first at {bad.nonzero()[0].tolist()}"


def layout(kind, M, S, dev, seed=7):
    """(index, rows_per_index, adapter of each row)"""
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        idx, per = torch.zeros(1, dtype=torch.int32), M
    elif kind == "groups":
        per = max(1, M // 5)
        idx = torch.randint(-1, S, ((M + per - 1) // per,), generator=g, dtype=torch.int32)
    elif kind == "rows":        # every row its own, in any order
        idx, per = torch.randint(-1, S, (M,), generator=g, dtype=torch.int32), 1
    elif kind == "ragged":      # requests of unequal lengths in order
        cuts = torch.sort(torch.randint(0, M + 1, (2 * S,), generator=g)).values
        who = torch.zeros(M, dtype=torch.int64)
        for c in cuts:
            who[int(c):] += 1
        idx, per = ((who * 5) % (S + 1) - 1).to(torch.int32), 1
    else:                       # "wild": entries outside [0, S) mean no adapter
        idx, per = torch.randint(-5, S + 5, (M,), generator=g, dtype=torch.int32), 1
    who = idx.to(torch.int64).repeat_interleave(per)[:M]
    return idx.to(dev), per, torch.where((who >= 0) & (who < S), who, torch.full_like(who, -1)).to(dev)


#        M     K     N    S   r   rows      extras
CASES = [
    (1, 8, 8, 1, 8, "one", ""),
    (8, 1280, 1280, 8, 16, "rows", "bias"),
    (33, 72, 40, 3, 24, "rows", ""),
    (77, 320, 320, 2, 16, "groups", "bias residual"),
    (300, 768, 640, 4, 8, "ragged", "half residual"),
    (514, 768, 640, 2, 40, "groups", "bias"),
    (1000, 640, 648, 5, 128, "ragged", "bias"),
    (2049, 320, 960, 7, 32, "wild", "residual"),
    (5003, 1280, 640, 7, 24, "ragged", "bias"),
    (40961, 320, 320, 3, 16, "groups", "bias"),       # whole-width tiles
    (33000, 256, 1280, 6, 64, "ragged", ""),          # 256 x 256 tiles
    (4100, 128, 512, 30, 8, "rows", "residual"),      # many adapters within a tile
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients_against_64_bits(dev, dtype, case):
    from mimo_amd import ops
    M, K, N, S, r, kind, extras = case
    a, w = rnd((M, K), dev, dtype, 1), rnd((N, K), dev, dtype, 2, K ** -0.5)
    down, up = rnd((S, r, K), dev, dtype, 3, K ** -0.5), rnd((S, N, r), dev, dtype, 4, r ** -0.5)
    scale = rnd((S,), dev, torch.float32, 5).abs() + 0.5
    bias = rnd((N,), dev, torch.float32, 6) if "bias" in extras else None
    res = rnd((M, N), dev, dtype if "half" in extras else torch.float32, 8) if "residual" in extras else None
    index, per, who = layout(kind, M, S, dev)
    kw = dict(rows_per_index=per, scale=scale)
    dout = rnd((M, N), dev, dtype, 9)
    for f32 in (False, True):
        out, low = ops.adapter_gemm(a, w, down, up, index, bias=bias, residual=res, out_f32=f32, want_low=True, **kw)
        assert out.dtype == (torch.float32 if f32 else dtype)
        assert torch.equal(out, ops.adapter_gemm(a, w, down, up, index, bias=bias, residual=res, out_f32=f32, **kw))
        val, bnd = reference(a, w, down, up, who, scale, bias, res, f32, None if f32 else dout)
        within("out", out, val["out"], bnd["out"])
        if not f32:
            grads = ops.adapter_gemm_backward(dout, a, w.t().contiguous(), down, up, index, low, **kw)
            for name, got in zip(("da", "ddown", "dup"), grads):
                within(name, got, val[name], bnd[name])
            again = ops.adapter_gemm_backward(dout, a, w.t().contiguous(), down, up, index, low, **kw)
            assert all(torch.equal(x, y) for x, y in zip(grads, again))
            none, dd, du = ops.adapter_gemm_backward(dout, a, w.t().contiguous(), down, up, index, low, want_da=False, **kw)
            assert none is None and torch.equal(dd, grads[1]) and torch.equal(du, grads[2])


@gpu
def test_strided_rows_no_scale_no_rows(dev):
    from mimo_amd import ops
    big, dbig = rnd((70, 3 * 64), dev, torch.float16, 1), rnd((70, 2 * 96), dev, torch.float16, 2)
    a, dout = big[:, 64:128], dbig[:, 96:]
    w, down, up = rnd((96, 64), dev, torch.float16, 3, 0.1), rnd((2, 8, 64), dev, torch.float16, 4, 0.1), rnd((2, 96, 8), dev, torch.float16, 5, 0.3)
    index = torch.tensor([1, 0, 1], dtype=torch.int32, device=dev)   # entries behind the last row are not read as rows
    out, low = ops.adapter_gemm(a, w, down, up, index, rows_per_index=40, want_low=True)
    who = index.long().repeat_interleave(40)[:70]
    val, bnd = reference(a, w, down, up, who, None, None, None, False, dout)
    within("out", out, val["out"], bnd["out"])
    for name, got in zip(("da", "ddown", "dup"), ops.adapter_gemm_backward(dout, a, w.t().contiguous(), down, up, index, low, rows_per_index=40)):
        within(name, got, val[name], bnd[name])
    row = a[:1].expand(5, 64)                                        # one row seen by five requests
    i5 = torch.tensor([0, 1, -1, 1, 0], dtype=torch.int32, device=dev)
    same = torch.equal(ops.adapter_gemm(row, w, down, up, i5), ops.adapter_gemm(row.contiguous(), w, down, up, i5))
    assert same
    out, low = ops.adapter_gemm(a[:0], w, down, up, index, want_low=True)
    da, ddown, dup = ops.adapter_gemm_backward(dout[:0], a[:0], w.t().contiguous(), down, up, index, low)
    assert out.shape == (0, 96) and da.shape == (0, 64) and not ddown.any() and not dup.any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_do_not_touch_each_other(dev, dtype):
    """A request whose adapter (or whose rows) holds NaN and infinities: the other requests of the same tiles get what they get
    without it, bit for bit, and so do their adapters' gradients."""
    from mimo_amd import ops
    M, K, N, S, r = 200, 128, 160, 3, 16
    a, w = rnd((M, K), dev, dtype, 1), rnd((N, K), dev, dtype, 2, 0.1)
    down, up = rnd((S, r, K), dev, dtype, 3, 0.1), rnd((S, N, r), dev, dtype, 4, 0.2)
    dout = rnd((M, N), dev, dtype, 5)
    index = torch.randint(0, S, (M,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(dev)
    mine = index != 1
    out, low = ops.adapter_gemm(a, w, down, up, index, want_low=True)
    grads = ops.adapter_gemm_backward(dout, a, w.t().contiguous(), down, up, index, low)
    d2, u2, a2, g2 = down.clone(), up.clone(), a.clone(), dout.clone()
    d2[1, 0, 0], u2[1, 5, 3], a2[~mine], g2[~mine] = float("nan"), float("inf"), float("nan"), float("-inf")
    out2, low2 = ops.adapter_gemm(a2, w, d2, u2, index, want_low=True)
    grads2 = ops.adapter_gemm_backward(g2, a2, w.t().contiguous(), d2, u2, index, low2)
    assert torch.equal(out[mine], out2[mine]) and torch.equal(low[mine], low2[mine]) and torch.equal(grads[0][mine], grads2[0][mine])
    for i in (0, 2):
        assert torch.equal(grads[1][i], grads2[1][i]) and torch.equal(grads[2][i], grads2[2][i])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N,r,per", [
    (3, 128, 160, 16, 1),          # the low-rank values inside the kernel for few rows
    (40, 128, 160, 16, 1),         # in front of it
    (61, 128, 160, 40, 7),         # ... by matrix tiles that several requests share
    (200, 128, 160, 16, 24),       # boundaries inside a tile of 32 rows and of 64
    (3000, 64, 320, 8, 100),
    (10300, 64, 1280, 16, 333),    # 256 x 256 tiles
    (33000, 64, 96, 24, 500),      # a wave per 32 rows
])
def test_requests_do_not_touch_each_other_in_any_kernel(dev, dtype, M, K, N, r, per):
    """As above, for each of the kernels that sizes select: a zero operand in place of a selection would let NaN through."""
    from mimo_amd import ops
    S = 3
    a, w = rnd((M, K), dev, dtype, 1), rnd((N, K), dev, dtype, 2, 0.1)
    down, up = rnd((S, r, K), dev, dtype, 3, 0.1), rnd((S, N, r), dev, dtype, 4, 0.2)
    dout = rnd((M, N), dev, dtype, 5)
    index = torch.tensor([(0, 1, 2, 1, -1)[i % 5] for i in range((M + per - 1) // per)], dtype=torch.int32, device=dev)
    mine = index.repeat_interleave(per)[:M] != 1
    wt = w.t().contiguous()
    d2, u2, a2, g2 = down.clone(), up.clone(), a.clone(), dout.clone()
    d2[1, 0, 0], u2[1, 5, 3], a2[~mine], g2[~mine] = float("nan"), float("inf"), float("nan"), float("-inf")
    for f32 in (False, True):
        out, low = ops.adapter_gemm(a, w, down, up, index, rows_per_index=per, want_low=True, out_f32=f32)
        out2, low2 = ops.adapter_gemm(a2, w, d2, u2, index, rows_per_index=per, want_low=True, out_f32=f32)
        assert torch.equal(out[mine], out2[mine]) and torch.equal(low[mine], low2[mine]), f32
    grads = ops.adapter_gemm_backward(dout, a, wt, down, up, index, low, rows_per_index=per)
    grads2 = ops.adapter_gemm_backward(g2, a2, wt, d2, u2, index, low2, rows_per_index=per)
    assert torch.equal(grads[0][mine], grads2[0][mine])
    for i in (0, 2):
        assert torch.equal(grads[1][i], grads2[1][i]) and torch.equal(grads[2][i], grads2[2][i])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,N,extras", [("ragged", 96, "bias"), ("groups", 160, "residual")])
def test_rows_so_far_apart_that_launches_are_cut(dev, dtype, kind, N, extras):
    """Rows 2^20 elements apart: 32-bit offsets reach 768 of them, so the tiles of 1100 rows go in two launches, the second with the
    index, the low-rank values, the result and the residual moved on."""
    from mimo_amd import ops
    M, K, S, r, far = 1100, 128, 4, 16, 1 << 20
    buf = torch.empty((M * far,), device=dev, dtype=dtype)
    a, dout = torch.as_strided(buf, (M, K), (far, 1), 0), torch.as_strided(buf, (M, N), (far, 1), 512)
    a.copy_(rnd((M, K), dev, dtype, 1)), dout.copy_(rnd((M, N), dev, dtype, 5))
    w, down, up = rnd((N, K), dev, dtype, 2, K ** -0.5), rnd((S, r, K), dev, dtype, 3, K ** -0.5), rnd((S, N, r), dev, dtype, 4, r ** -0.5)
    scale = rnd((S,), dev, torch.float32, 6).abs() + 0.5
    bias = rnd((N,), dev, torch.float32, 7) if extras == "bias" else None
    res = rnd((M, N), dev, torch.float32, 8) if extras == "residual" else None
    index, per, who = layout(kind, M, S, dev)
    kw = dict(rows_per_index=per, scale=scale)
    for f32 in (False, True):
        out, low = ops.adapter_gemm(a, w, down, up, index, bias=bias, residual=res, out_f32=f32, want_low=True, **kw)
        val, bnd = reference(a, w, down, up, who, scale, bias, res, f32, None if f32 else dout)
        within("out", out, val["out"], bnd["out"])
        if not f32:
            for name, got in zip(("da", "ddown", "dup"), ops.adapter_gemm_backward(dout, a, w.t().contiguous(), down, up, index, low, **kw)):
                within(name, got, val[name], bnd[name])


@gpu
@pytest.mark.parametrize("M", [3, 40, 900])
def test_low_rank_values_up_to_the_largest_fp16_and_beyond(dev, M):
    """u and t up to 65504: right.  Beyond it: the rows concerned are infinite or NaN and the others are right; no finite number is wrong."""
    from mimo_amd import ops
    K, N, r = 64, 96, 8
    w, wt = torch.zeros((N, K), device=dev, dtype=H), torch.zeros((K, N), device=dev, dtype=H)
    a, dout = (torch.ones((M, n), device=dev, dtype=H) for n in (K, N))
    down, up = torch.full((1, r, K), 2.0 ** -10, device=dev, dtype=H), torch.full((1, N, r), 2.0 ** -10, device=dev, dtype=H)
    index = torch.zeros(1, dtype=torch.int32, device=dev)

    def run(size, back):   # every u is `size`, every t is `back`
        out, low = ops.adapter_gemm(size * 2.0 ** 4 * a, w, down, up, index, rows_per_index=M, want_low=True)
        return out, low, *ops.adapter_gemm_backward(back * (2.0 ** 10 / N) * dout, a, wt, down, up, index, low, rows_per_index=M)
    out, low, da, ddown, dup = run(4094.0, 384.0)   # (inputs within fp16 too)
    assert torch.equal(out, torch.full_like(out, 4094.0 * r * 2.0 ** -10)) and torch.isfinite(ddown).all() and torch.isfinite(dup).all()
    big = 2.0 ** 5      # the same with weights and adapters 2^5 larger: u = 131008, t = 12288
    down, up = down * big, up * big
    out, low, da, ddown, dup = run(4094.0, 384.0)
    assert not torch.isfinite(out).any() and torch.isfinite(ddown).all()
    a2, a3 = a.clone(), 4094.0 * 2.0 ** 4 * a
    a3[1:] = a2[1:]
    out, low = ops.adapter_gemm(a3, w, down, up, index, rows_per_index=M, want_low=True)
    assert not torch.isfinite(out[0]).any() and torch.equal(out[1:], torch.full_like(out[1:], K * 2.0 ** -5 * r * 2.0 ** -5))
    g = dout.clone()
    g[0] = 384.0 * 2.0 ** 10 / N * 8    # t = 98304 in row 0, 3 elsewhere
    _, low = ops.adapter_gemm(a, w, down, up, index, rows_per_index=M, want_low=True)
    da, ddown, dup = ops.adapter_gemm_backward(g, a, wt, down, up, index, low, rows_per_index=M)
    assert not torch.isfinite(da[0]).any() and torch.equal(da[1:], torch.full_like(da[1:], N * 2.0 ** -5 * r * 2.0 ** -5))
    assert not torch.isfinite(ddown).any() and torch.isfinite(dup).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("M,r", [(1, 8), (3, 40), (4, 64), (4, 128), (9, 16), (70, 16), (2100, 16)])
def test_low_holds_the_low_rank_values_afterwards(dev, dtype, split, M, r):
    """What the C entry promises of `low`, whichever kernel the number of rows and the rank select: the rows' values rounded once, or
    value and remainders, and zeros for a row without an adapter."""
    from mimo_amd import lib, ops
    K, N, S = 96, 80, 3
    a, w = rnd((M, K), dev, dtype, 1), rnd((N, K), dev, dtype, 2, 0.1)
    down, up, scale = rnd((S, r, K), dev, dtype, 3, 0.1), rnd((S, N, r), dev, dtype, 4, 0.1), rnd((S,), dev, torch.float32, 5).abs() + 0.5
    index, per, who = layout("rows", M, S, dev)
    planes = ops.LOW_PLANES[dtype] if split else 1
    low, out = torch.full((M, planes * r), float("nan"), device=dev, dtype=dtype), torch.empty((M, N), device=dev, dtype=dtype)
    p = lib.AdapterParams(down.data_ptr(), up.data_ptr(), scale.data_ptr(), index.data_ptr(), per, S, r)
    lib.call("mimo_adapter_gemm", lib.F16 if dtype == torch.float16 else lib.BF16, a.data_ptr(), K, w.data_ptr(), out.data_ptr(), N, M, N, K,
             None, None, 0, 0, ctypes.byref(p), low.data_ptr(), split, torch.cuda.current_stream().cuda_stream)
    val, size = (torch.zeros((M, r), dtype=torch.float64, device=dev) for _ in range(2))
    for i in range(S):
        at = who == i
        val[at] = float(scale[i]) * a[at].double() @ down[i].double().t()
        size[at] = float(scale[i]) * a[at].double().abs() @ down[i].double().abs().t()
    u, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    got = low.double().reshape(M, planes, r).sum(1)
    within("low", got, val, acc(K) * size + (u ** planes if split else u) * val.abs() * 1.01 + tiny)


@gpu
def test_gradient_against_differences(dev):
    """The directional derivative of sum(out g) along a step of a, down and up: the formula is bilinear in down and up and linear in
    a, so one central difference in 64 bits is exact."""
    from mimo_amd import ops
    M, K, N, S, r = 90, 64, 72, 3, 8
    dt = torch.float16
    a, w = rnd((M, K), dev, dt, 1), rnd((N, K), dev, dt, 2, 0.1)
    down, up, g = rnd((S, r, K), dev, dt, 3, 0.1), rnd((S, N, r), dev, dt, 4, 0.3), rnd((M, N), dev, dt, 5)
    scale = rnd((S,), dev, torch.float32, 6).abs() + 0.5
    index, per, who = layout("ragged", M, S, dev)
    _, low = ops.adapter_gemm(a, w, down, up, index, scale=scale, want_low=True)
    grads = ops.adapter_gemm_backward(g, a, w.t().contiguous(), down, up, index, low, scale=scale)
    _, bnd = reference(a, w, down, up, who, scale, None, None, False, g)
    args = [x.double() for x in (a, down, up)]

    def f(x):
        y = x[0] @ w.double().t()
        for i in range(S):
            at = (who == i).nonzero()[:, 0]
            y[at] += float(scale[i]) * (x[0][at] @ x[1][i].t()) @ x[2][i].t()
        return float((y * g.double()).sum())

    for i, (name, got) in enumerate(zip(("da", "ddown", "dup"), grads)):
        step = rnd(got.shape, dev, torch.float64, 30 + i)
        ends = []
        for sign in (1, -1):
            x = list(args)
            x[i] = x[i] + sign * step
            ends.append(f(x))
        off = float((bnd[name] * step.abs()).sum())
        assert abs(float((got.double() * step).sum()) - (ends[0] - ends[1]) / 2) <= off + 1e-9 * abs(ends[0])


@gpu
def test_other_streams_and_graphs(dev):
    from mimo_amd import ops
    shapes = [(8, 320, 320, 4, 16, "rows"), (700, 128, 320, 3, 32, "ragged")]
    data = []
    for M, K, N, S, r, kind in shapes:
        index, per, _ = layout(kind, M, S, dev)
        w = rnd((N, K), dev, torch.bfloat16, 2, 0.1)
        data.append((rnd((M, K), dev, torch.bfloat16, 1), w, w.t().contiguous(), rnd((S, r, K), dev, torch.bfloat16, 3, 0.1),
                     rnd((S, N, r), dev, torch.bfloat16, 4, 0.3), index, rnd((M, N), dev, torch.bfloat16, 5)))

    def step(i, a):
        _, w, wt, down, up, index, dout = data[i]
        out, low = ops.adapter_gemm(a, w, down, up, index, want_low=True)
        return (out,) + ops.adapter_gemm_backward(dout, a, wt, down, up, index, low)

    want = [step(i, data[i][0]) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i, data[i][0])
    torch.cuda.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(x, y))
    for i in range(2):
        a = data[i][0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(i, a)
        for n in range(4):
            a.copy_(rnd(a.shape, dev, a.dtype, 50 + n))
            ref = step(i, a)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(ref, res)), (i, n)


# ---- refusals and packing: the host --------------------------------------------------------------------------------------------
H = torch.float16


@pytest.mark.parametrize("change,why", [
    (dict(), "device tensor"),
    (dict(a=torch.zeros(6, 16)), "float16 or bfloat16"),
    (dict(a=torch.zeros(6, 24, dtype=H)), "fit together"),
    (dict(w=torch.zeros(16, 24, dtype=H)), "fit together"),
    (dict(up=torch.zeros(2, 24, 16, dtype=H)), "fit together"),
    (dict(up=torch.zeros(3, 24, 8, dtype=H)), "fit together"),
    (dict(down=torch.zeros(2, 4, 16, dtype=H), up=torch.zeros(2, 24, 4, dtype=H)), "rank 4"),
    (dict(down=torch.zeros(2, 136, 16, dtype=H), up=torch.zeros(2, 24, 136, dtype=H)), "rank 136"),
    (dict(w=torch.zeros(24, 16)), "float32"),
    (dict(w=torch.zeros(16, 24, dtype=H).t()), "contiguous"),
    (dict(a=torch.zeros(6, 20, dtype=H)[:, :16]), "16-byte"),
    (dict(a=torch.zeros(16, 6, dtype=H).t()), "last axis"),
    (dict(index=torch.zeros(6)), "index"),
    (dict(index=torch.zeros(5, dtype=torch.int32)), "index"),
    (dict(rows_per_index=0), "rows_per_index"),
    (dict(rows_per_index=2, index=torch.zeros(2, dtype=torch.int32)), "index"),
    (dict(scale=torch.zeros(3)), "scale"),
    (dict(scale=torch.zeros(2, dtype=torch.float64)), "scale"),
])
def test_refusals(change, why):
    from mimo_amd import lib, ops
    x = dict(a=torch.zeros(6, 16, dtype=H), w=torch.zeros(24, 16, dtype=H), down=torch.zeros(2, 8, 16, dtype=H),
             up=torch.zeros(2, 24, 8, dtype=H), index=torch.zeros(6, dtype=torch.int32))
    x.update(change)
    with pytest.raises(lib.MimoHipError, match=why):
        ops.adapter_gemm(**x)


def test_c_entry_refuses_what_it_cannot_run():
    from mimo_amd import lib
    L = lib.load()

    def params(**kw):
        p = lib.AdapterParams(4096, 4096, None, 4096, 1, 2, 16)
        for n, v in kw.items():
            setattr(p, n, v)
        return p

    def fwd(p=None, A=4096, lda=64, ldo=64, M=8, N=64, K=64, ldr=0, res=None, flags=0, low=4096, split=1, dtype=lib.F16):
        return L.mimo_adapter_gemm(dtype, A, lda, 4096, 4096, ldo, M, N, K, None, res, ldr, flags, ctypes.byref(p or params()), low, split, None)

    def bwd(p=None, M=8, N=64, K=64, ws=4096, nb=1 << 30, dA=4096, Wt=4096, ldy=64):
        return L.mimo_adapter_gemm_backward(lib.F16, 4096, ldy, 4096, 64, Wt, dA, 64, M, N, K, ctypes.byref(p or params()), 4096, 4096, 4096,
                                            ws, nb, None)

    for kw in (dict(down=None), dict(up=4100), dict(index=None), dict(index=4098), dict(rows_per_index=0), dict(count=0), dict(count=70000),
               dict(rank=0), dict(rank=12), dict(rank=136)):
        assert fwd(params(**kw)) == -1 and bwd(params(**kw)) == -1, kw
        assert L.mimo_adapter_gemm_backward_workspace(lib.F16, ctypes.byref(params(**kw)), 8, 64, 64) == 0
    for kw in (dict(M=0), dict(N=60), dict(K=12), dict(N=1 << 16, K=1 << 16)):
        assert fwd(**kw) == -1 and bwd(**kw) == -1, kw
    assert fwd(A=None) == -1 and fwd(A=4104) == -1 and fwd(lda=68) == -1 and fwd(ldo=66) == -1 and fwd(res=4096, ldr=2) == -1
    assert fwd(flags=lib.EPI_SILU) == -1 and fwd(flags=lib.EPI_OUT_F32, split=0) == -1 and fwd(low=None) == -1
    assert fwd(dtype=9) == -2
    assert bwd(ws=None) == -1 and bwd(nb=64) == -1 and bwd(Wt=None) == -1 and bwd(ldy=4) == -1


def test_refuses_rows_and_widths_behind_32_bit_offsets():
    from mimo_amd import lib, ops
    x = dict(a=torch.zeros(6, 16, dtype=H), w=torch.zeros(24, 16, dtype=H), down=torch.zeros(2, 8, 16, dtype=H),
             up=torch.zeros(2, 24, 8, dtype=H), index=torch.zeros(6, dtype=torch.int32))
    far = lambda n, dt=H: torch.empty_strided((6, n), ((1 << 20) + 8, 1), dtype=dt)
    with pytest.raises(lib.MimoHipError, match="elements apart"):
        ops.adapter_gemm(**{**x, "a": far(16)})
    for t in (far(24), far(24, torch.float32)):
        with pytest.raises(lib.MimoHipError, match="elements apart"):
            ops._pitch_ok(t, "residual")
    ops._pitch_ok(far(24)[:1], "residual")
    n = 1 << 20
    wide = dict(a=torch.zeros(6, 8, dtype=H), w=torch.zeros(n, 8, dtype=H), down=torch.zeros(1, 8, 8, dtype=H), up=torch.zeros(1, n, 8, dtype=H),
                index=x["index"])
    with pytest.raises(lib.MimoHipError, match="beyond what"):
        ops.adapter_gemm(**wide)
    L = lib.load()
    p = lib.AdapterParams(4096, 4096, None, 4096, 1, 2, 16)
    call = lambda N=64, K=64, lda=64, ldo=64, res=None, ldr=64: L.mimo_adapter_gemm(
        lib.F16, 4096, lda, 4096, 4096, ldo, 8, N, K, None, res, ldr, 0, ctypes.byref(p), 4096, 1, None)
    back = lambda ldy=64, ldda=64: L.mimo_adapter_gemm_backward(lib.F16, 4096, ldy, 4096, 64, 4096, 4096, ldda, 8, 64, 64, ctypes.byref(p), 4096,
                                                                4096, 4096, 4096, 1 << 30, None)
    far = (1 << 20) + 8
    assert call(N=n, ldo=n) == call(K=n, lda=n) == call(lda=far) == call(ldo=far) == call(ldo=-8) == call(res=4096, ldr=far) == -1
    assert call(res=4096, ldr=-8) == back(ldy=far) == back(ldda=far) == back(ldda=-8) == -1


def test_pack_adapters_pads_and_stacks():
    from mimo_amd.packing import pack_adapters
    g = torch.Generator().manual_seed(0)
    raw = [(torch.randn(r, 24, generator=g), torch.randn(40, r, generator=g), al) for r, al in ((4, 8.0), (12, None), (1, 0.5))]
    p = pack_adapters(raw, torch.float32)
    assert p["down"].shape == (3, 16, 24) and p["up"].shape == (3, 40, 16) and p["scale"].tolist() == [2.0, 1.0, 0.5]
    for i, (d, u, _) in enumerate(raw):
        assert torch.allclose(p["up"][i] @ p["down"][i], u @ d, atol=1e-5)
