"""Cross attention to encoder states of another length (ops.cross_attention / cross_attention_backward): the HIP kernels against
the formulas in 64 bits, element by element, under bounds that count the kernels' own roundings.

With u = eps / 2 of the operand type: out = (sum_k half(p) v) / l rounds every p once and the result once, so
|error| <= u (sum_k p |v| / l + |out|); lse, delta and every sum are fp32, whose errors enter through the scores:
ds = d 2^-24 scale max sum_c |q_c k_c| (a dot product of d terms), i.e. a factor 1 +- 2 ds on every p.  Values of p or dS below
the normal range of fp16 are off by at most 2^-25 absolutely.  The gradients likewise: dS rounds once, delta is taken from the
rounded output (|d delta| <= u sum |dO o|) unless few keys count, the result rounds once."""
import ctypes

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


def keep_of(Be, Nk, kv_len, mask, dev):
    keep = torch.ones((Be, Nk), dtype=torch.bool, device=dev)
    if kv_len is not None:
        keep &= torch.arange(Nk, device=dev)[None] < kv_len[:, None].clamp(0, Nk)
    if mask is not None:
        keep &= mask.bool()
    return keep


def reference(q, k, v, heads, kvh, keep, scale, dout=None):
    """(values, bounds), dicts of fp64 tensors: out, lse and, with dout, dq, dk, dv — from the formulas."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    B, Nq, C = q.shape
    Be, Nk, _ = k.shape
    d, rep, hg = C // heads, B // Be, heads // kvh
    zero = ~keep[..., None]
    # [Be, kvh, rep, Nq, hg, d] queries; [Be, kvh, 1, 1, Nk, d] keys
    Q = q.double().reshape(Be, rep, Nq, kvh, hg, d).permute(0, 3, 1, 2, 4, 5).reshape(Be, kvh, -1, d)
    K = k.double().masked_fill(zero, 0).reshape(Be, Nk, kvh, d).transpose(1, 2)
    V = v.double().masked_fill(zero, 0).reshape(Be, Nk, kvh, d).transpose(1, 2)

    def rows(x):   # [Be, kvh, rep Nq hg, d] -> [B, Nq, C]
        return x.reshape(Be, kvh, rep, Nq, hg, d).permute(0, 2, 3, 1, 4, 5).reshape(B, Nq, C)

    def keys(x):
        return x.transpose(1, 2).reshape(Be, Nk, kvh * d)

    see = keep[:, None, None, :]
    S = (Q @ K.transpose(2, 3) * scale).masked_fill(~see, float("-inf"))
    lse = torch.logsumexp(S, -1, keepdim=True)
    P = torch.where(see.expand_as(S), torch.exp(S - lse.masked_fill(lse == float("-inf"), 0)), torch.zeros_like(S))
    slack = 2 * (d * 2.0 ** -24 * scale * float((Q.abs() @ K.abs().transpose(2, 3)).max()) if Nk else 0.0) + 2e-6
    O = P @ V
    val = dict(out=rows(O), lse=lse.reshape(Be, kvh, rep, Nq, hg).permute(0, 2, 1, 4, 3).reshape(B, heads, Nq))
    A = P @ V.abs()
    bnd = dict(out=rows((u + slack) * A * 1.01 + u * O.abs() + tiny * (1 + V.abs().sum(2, keepdim=True))),
               lse=(slack + 2.0 ** -23 * val["lse"].abs()).masked_fill(val["lse"] == float("-inf"), 0))
    if dout is None:
        return val, bnd
    dO = dout.double().reshape(Be, rep, Nq, kvh, hg, d).permute(0, 3, 1, 2, 4, 5).reshape(Be, kvh, -1, d)
    dP = dO @ V.transpose(2, 3)
    delta = (dO * O).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    val.update(dq=rows(scale * dS @ K), dk=keys(scale * dS.transpose(2, 3) @ Q), dv=keys(P.transpose(2, 3) @ dO))
    # delta comes from the output as it was stored: its own bound, times |dO|
    E = (u + slack) * A * 1.01 + u * O.abs() + tiny * (1 + V.abs().sum(2, keepdim=True))
    eS = u * dS.abs() + P * (slack * (dP.abs() + delta.abs()) + (dO.abs() * E).sum(-1, keepdim=True) +
                             d * 2.0 ** -24 * (dO.abs() @ V.abs().transpose(2, 3) + (dO * O).abs().sum(-1, keepdim=True))) * (1 + u) + tiny
    eS = eS * see
    bnd.update(dq=rows(scale * eS @ K.abs()) * 1.01 + u * val["dq"].abs() + tiny,
               dk=keys(scale * eS.transpose(2, 3) @ Q.abs()) * 1.01 + (u + 1e-6) * val["dk"].abs() + tiny,
               dv=keys((((u + slack) * P + tiny) * see).transpose(2, 3) @ dO.abs()) * 1.01 + (u + 1e-6) * val["dv"].abs() + tiny)
    return val, bnd


def within(name, got, val, bnd):
    inf = val == float("-inf")
    assert torch.equal(inf, got.double() == float("-inf")), name
    err = (got.double() - val).masked_fill(inf, 0).abs()
    bad = ~(err <= bnd)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()}, worst error / bound {float((err / bnd.clamp_min(1e-300))[bad].max()):.3g}, " \
                          f"first at {bad.nonzero()[0].tolist()}"


#        B  Be  Nq   Nk  heads kvh  d   keys
CASES = [
    (1, 1, 1, 1, 1, 1, 8, "full"),
    (2, 1, 5, 3, 2, 2, 16, "full"),
    (6, 2, 33, 77, 8, 8, 40, "lengths"),
    (4, 2, 64, 257, 8, 8, 80, "mask"),
    (3, 3, 130, 96, 3, 3, 24, "both"),
    (4, 1, 9, 31, 6, 2, 96, "lengths"),
    (2, 2, 65, 64, 4, 4, 48, "full"),
    (16, 8, 7, 33, 4, 2, 72, "mask"),
    (2, 2, 100, 700, 2, 2, 160, "lengths"),       # streamed, several query tiles
    (8, 4, 1, 1000, 8, 1, 64, "lengths"),         # single tokens, keys cut into parts
    (3, 3, 2, 4097, 4, 4, 128, "mask"),           # ... and a mask
    (5, 5, 1, 12345, 2, 2, 32, "full"),
    (2, 2, 300, 2050, 2, 1, 56, "both"),
    (24, 3, 255, 16, 8, 8, 160, "lengths"),
    (1, 1, 2500, 40, 8, 8, 40, "full"),           # several tiles per wave, parts of the rows in the backward
]


def make(case, dev, dtype, garbage=True):
    B, Be, Nq, Nk, heads, kvh, d, keys = case
    kv = rnd((Be, Nk, 2 * kvh * d), dev, dtype, 2)
    q = rnd((B, Nq, heads * d), dev, dtype, 1)
    k, v = kv[..., :kvh * d], kv[..., kvh * d:]
    kv_len = mask = None
    g = torch.Generator().manual_seed(5)
    if keys in ("lengths", "both"):
        kv_len = torch.randint(0, Nk + 1, (Be,), generator=g)
        kv_len[0] = Nk - 1
        if Be > 1:
            kv_len[-1] = 0
        kv_len = kv_len.to(torch.int32).to(dev)
    if keys in ("mask", "both"):
        mask = torch.rand((Be, Nk), generator=g) < 0.6
        if Be > 1:
            mask[1] = False
        mask = mask.to(dev)
    keep = keep_of(Be, Nk, kv_len, mask, dev)
    if garbage:   # what stands at keys that do not count must not matter
        junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min], device=dev, dtype=dtype)
        fill = junk[torch.arange(kv.numel(), device=dev).reshape(kv.shape) % 4]
        kv.copy_(torch.where(keep[..., None], kv, fill))
    return q, k, v, dict(kv_heads=kvh, kv_len=kv_len, mask=mask), keep


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients_against_64_bits(dev, dtype, case):
    from mimo_amd import ops
    q, k, v, kw, keep = make(case, dev, dtype)
    heads, d = case[4], case[6]
    dout = rnd(q.shape, dev, dtype, 3)
    out, lse = ops.cross_attention(q, k, v, heads, want_lse=True, **kw)
    assert torch.equal(out, ops.cross_attention(q, k, v, heads, **kw))
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse, heads, **kw)
    val, bnd = reference(q, k, v, heads, kw["kv_heads"], keep, d ** -0.5, dout)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + grads):
        assert got.dtype == (torch.float32 if name == "lse" else dtype) and got.shape == val[name].shape
        within(name, got, val[name], bnd[name])
    again = ops.cross_attention_backward(dout, q, k, v, out, lse, heads, **kw)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))   # no atomics: the same bits


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_broadcast_operands(dev, dtype):
    """q inside a fused projection, a transposed batch axis, one query row seen by every image (stride 0), a scale of one's own."""
    from mimo_amd import ops
    heads, d, Nq, Nk = 4, 40, 37, 50
    C = heads * d
    qkv = rnd((6, Nq, 3 * C), dev, dtype, 1)
    kv = rnd((Nk, 3, 2 * C), dev, dtype, 2).transpose(0, 1)
    big = rnd((Nq, 6, C + 8), dev, dtype, 3)
    dout = big[..., :C].transpose(0, 1)
    keep = keep_of(3, Nk, None, None, dev)
    for q in (qkv[..., C:2 * C], qkv[:1, :, :C].expand(6, Nq, C)):
        out, lse = ops.cross_attention(q, kv[..., :C], kv[..., C:], heads, scale=0.3, want_lse=True)
        grads = ops.cross_attention_backward(dout, q, kv[..., :C], kv[..., C:], out, lse, heads, scale=0.3)
        val, bnd = reference(q, kv[..., :C], kv[..., C:], heads, heads, keep, 0.3, dout)
        for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + grads):
            within(name, got, val[name], bnd[name])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Nq,Nk,heads,kvh,d,live", [(600, 2, 4, 4, 40, 2), (600, 77, 4, 2, 40, 3), (300, 257, 4, 4, 160, 5), (500, 64, 4, 4, 64, 20),
                                                    (300, 300, 2, 2, 160, 30)])
def test_gradients_of_few_keys(dev, dtype, Nq, Nk, heads, kvh, d, live):
    """Where few keys share a row dS is a small difference of P dP and P delta, and a delta taken from the rounded output would double
    dQ's error.  What is left are two roundings, dS's and the result's, each uniform within half a step: 0.425 u of the value in the
    mean square (1 / sqrt(3), mantissas spread evenly in their logarithm), independent of each other; 15 % for the sample."""
    from mimo_amd import ops
    q, kv = rnd((2, Nq, heads * d), dev, dtype, 11), rnd((2, Nk, 2 * kvh * d), dev, dtype, 12)
    k, v, dout = kv[..., :kvh * d], kv[..., kvh * d:], rnd((2, Nq, heads * d), dev, dtype, 13)
    kv_len = mask = None
    keep = torch.zeros((2, Nk), dtype=torch.bool, device=dev)
    if live < Nk:   # row 0: anywhere, by the mask; row 1: in front, by the mask
        keep[0, torch.randperm(Nk, generator=torch.Generator().manual_seed(4))[:live].to(dev)] = True
        keep[1, :live] = True
        mask = keep
    else:
        keep[:] = True
    out, lse = ops.cross_attention(q, k, v, heads, kv_heads=kvh, mask=mask, want_lse=True)
    val, _ = reference(q, k, v, heads, kvh, keep, d ** -0.5, dout)
    u, tiny, hg = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0, heads // kvh
    split = lambda x, n: x.double().reshape(2, -1, n, d).transpose(1, 2)
    Q, G, K, V = split(q, heads), split(dout, heads), split(k, kvh).repeat_interleave(hg, 1), split(v, kvh).repeat_interleave(hg, 1)
    P = (Q @ K.transpose(2, 3) * d ** -0.5).masked_fill(~keep[:, None, None, :], float("-inf")).softmax(-1)
    dP = G @ V.transpose(2, 3)
    dS2 = (P * (dP - (P * dP).sum(-1, keepdim=True))).square() * (0.425 * u) ** 2 + tiny ** 2 * keep[:, None, None, :]
    for name, got, from_dS in zip(("dq", "dk"), ops.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kvh, mask=mask),
                                  (dS2 @ K.square(), dS2.transpose(2, 3) @ Q.square())):
        left = float((from_dS.sum() / d + val[name].square().sum() * (0.425 * u) ** 2 + tiny ** 2 * got.numel()).sqrt())
        off = float((got.double() - val[name]).norm())
        assert off <= 1.15 * left, (name, off, left)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Nk,d", [(77, 8), (64, 16), (83, 32)])
def test_query_gradient_of_narrow_heads(dev, dtype, Nk, d):
    """Heads up to 32 wide: dS is not rounded for dQ (its remainder takes part), what is left are the result's rounding and delta's,
    from the rounded output: 0.425 u of the values in the mean square, 15 % for the sample."""
    from mimo_amd import ops
    B, Nq, heads = 2, 700, 4
    q, k, v, dout = (rnd((B, n, heads * d), dev, dtype, 20 + i) for i, n in enumerate((Nq, Nk, Nk, Nq)))
    out, lse = ops.cross_attention(q, k, v, heads, want_lse=True)
    dq = ops.cross_attention_backward(dout, q, k, v, out, lse, heads)[0]
    val, _ = reference(q, k, v, heads, heads, torch.ones((B, Nk), dtype=torch.bool, device=dev), d ** -0.5, dout)
    r, tiny = 0.425 * torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    split = lambda x: x.double().reshape(B, -1, heads, d).transpose(1, 2)
    Q, K, G, O = split(q), split(k), split(dout), split(val["out"])
    PK = (Q @ K.transpose(2, 3) * d ** -0.5).softmax(-1) @ K
    from_delta = ((G * O).square().sum(-1, keepdim=True) * PK.square()).sum() / d
    left = float((r * r * (val["dq"].square().sum() + from_delta) + tiny ** 2 * dq.numel()).sqrt())
    off = float((dq.double() - val["dq"]).norm())
    assert off <= 1.15 * left, (off, left)


@gpu
def test_gradient_against_differences(dev):
    """The directional derivative of sum(out w) along a step of q, k and v: differences of the formula in 64 bits."""
    from mimo_amd import ops
    case = (4, 2, 20, 45, 4, 2, 40, "both")
    q, k, v, kw, keep = make(case, dev, torch.float16, garbage=False)
    w = rnd(q.shape, dev, torch.float16, 9)
    out, lse = ops.cross_attention(q, k, v, 4, want_lse=True, **kw)
    grads = ops.cross_attention_backward(w, q, k, v, out, lse, 4, **kw)
    args = [x.double() for x in (q, k, v)]
    for i, g in enumerate(grads):
        step = rnd(g.shape, dev, torch.float64, 20 + i)
        h = 1e-5

        def f(t):
            x = list(args)
            x[i] = x[i] + t * step
            B, Nq, C = q.shape
            Q = x[0].reshape(2, 2, Nq, 2, 2, 40).permute(0, 3, 1, 2, 4, 5).reshape(2, 2, -1, 40)
            K, V = (y.reshape(2, 45, 2, 40).transpose(1, 2) for y in x[1:])
            S = (Q @ K.transpose(2, 3) * 40 ** -0.5).masked_fill(~keep[:, None, None], -1e300)
            o = (torch.softmax(S, -1) * keep[:, None, None]) @ V
            return float((o * w.double().reshape(2, 2, Nq, 2, 2, 40).permute(0, 3, 1, 2, 4, 5).reshape(2, 2, -1, 40)).sum())

        diff = (f(h) - f(-h)) / (2 * h)
        _, bnd = reference(q, k, v, 4, 2, keep, 40 ** -0.5, w)
        off = float((bnd[("dq", "dk", "dv")[i]] * step.abs()).sum())   # every element at its bound, all of one sign
        assert abs(float((g.double() * step).sum()) - diff) <= off + 1e-6 * abs(diff)


@gpu
def test_no_keys_no_queries(dev):
    from mimo_amd import ops
    q = rnd((4, 6, 64), dev, torch.float16, 1)
    none = torch.empty((2, 0, 64), device=dev, dtype=torch.float16)
    out, lse = ops.cross_attention(q, none, none, 2, want_lse=True)
    assert not out.any() and (lse == float("-inf")).all()
    dq, dk, dv = ops.cross_attention_backward(q, q, none, none, out, lse, 2)
    assert not dq.any() and dk.shape == none.shape and dv.shape == none.shape
    k = rnd((2, 5, 64), dev, torch.float16, 2)
    for empty in (q[:, :0], q[:0]):
        out, lse = ops.cross_attention(empty, k, k, 2, want_lse=True)
        assert out.shape == empty.shape
        dq, dk, dv = ops.cross_attention_backward(empty, empty, k, k, out, lse, 2)
        assert dq.shape == empty.shape and not dk.any() and not dv.any()
    # lengths outside [0, Nk] count as the nearest end
    a = ops.cross_attention(q, k, k, 2, kv_len=torch.tensor([-3, 99], dtype=torch.int32, device=dev))
    b = ops.cross_attention(q, k, k, 2, kv_len=torch.tensor([0, 5], dtype=torch.int32, device=dev))
    assert torch.equal(a, b) and not a[:2].any()


@gpu
def test_rows_far_apart_in_memory(dev):
    """Row strides whose offsets pass 2^31 elements and 2^32 bytes."""
    from mimo_amd import ops
    far, C = 1 << 30, 64
    buf = torch.empty((2 * far + 4096,), device=dev, dtype=torch.float16)
    q = torch.as_strided(buf, (1, 3, C), (0, far, 1), 0)
    k = torch.as_strided(buf, (1, 3, C), (0, far, 1), 128)
    v = torch.as_strided(buf, (3, 1, C), (far, 0, 1), 256).transpose(0, 1)
    for i, t in enumerate((q, k, v)):
        t.copy_(rnd(t.shape, dev, torch.float16, i))
    out, lse = ops.cross_attention(q, k, v, 2, want_lse=True)
    grads = ops.cross_attention_backward(q, q, k, v, out, lse, 2)
    c = [x.contiguous() for x in (q, k, v)]
    out2, lse2 = ops.cross_attention(*c, 2, want_lse=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.cross_attention_backward(c[0], *c, out2, lse2, 2)))


@gpu
def test_other_streams_and_graphs(dev):
    """Two calls at once on two streams, and a captured forward + backward replayed with new inputs between eager calls."""
    from mimo_amd import ops
    cases = [(8, 4, 1, 1000, 8, 1, 64, "lengths"), (4, 2, 200, 100, 4, 4, 40, "mask")]
    data = [make(c, dev, torch.bfloat16) for c in cases]

    def step(i, q):
        _, k, v, kw, _ = data[i]
        out, lse = ops.cross_attention(q, k, v, cases[i][4], want_lse=True, **kw)
        return (out,) + ops.cross_attention_backward(q, q, k, v, out, lse, cases[i][4], **kw)

    want = [step(i, data[i][0]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i, data[i][0])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for i in range(2):
        q = data[i][0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(i, q)
        for n in range(4):
            q.copy_(rnd(q.shape, dev, q.dtype, 50 + n))
            ref = step(i, q)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(ref, res)), (i, n)


# ---- refusals: decided on the host, before any launch -------------------------------------------------------------------------
def _host(**kw):
    f = lambda *s: torch.zeros(s, dtype=torch.float16)
    a = dict(q=f(4, 6, 64), k=f(2, 5, 64), v=f(2, 5, 64), heads=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,why", [
    (dict(), "device tensor"),
    (dict(heads=3), "heads"),
    (dict(heads=16), "head width"),
    (dict(kv_heads=3), "key heads"),
    (dict(kv_heads=1), "encoder rows, keys"),
    (dict(k=torch.zeros(3, 5, 64, dtype=torch.float16), v=torch.zeros(3, 5, 64, dtype=torch.float16)), "4 images over 3"),
    (dict(v=torch.zeros(2, 4, 64, dtype=torch.float16)), "encoder rows, keys"),
    (dict(k=torch.zeros(2, 5, 64)), "float32"),
    (dict(q=torch.zeros(4, 6, 64)), "float16 or bfloat16"),
    (dict(q=torch.zeros(4, 64, dtype=torch.float16)), "batch, tokens, channels"),
    (dict(q=torch.zeros(4, 64, 6, dtype=torch.float16).transpose(1, 2)), "last axis"),
    (dict(q=torch.zeros(4, 6, 66, dtype=torch.float16)[..., :64]), "16-byte"),
    (dict(k=torch.zeros(2, 5, 72, dtype=torch.float16)[..., 4:68]), "16-byte"),
    (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(kv_len=torch.zeros(2)), "kv_len"),
    (dict(kv_len=torch.zeros(4, dtype=torch.int32)), "kv_len"),
    (dict(mask=torch.zeros(2, 5)), "mask"),
    (dict(mask=torch.zeros(5, 2, dtype=torch.bool).t()), "mask"),
    (dict(mask=torch.zeros(2, 6, dtype=torch.bool)), "mask"),
])
def test_refusals(change, why):
    from mimo_amd import lib, ops
    a = _host(**change)
    with pytest.raises(lib.MimoHipError, match=why):
        ops.cross_attention(**a)
    a["out"] = torch.zeros_like(a["q"])
    with pytest.raises(lib.MimoHipError, match=why):
        ops.cross_attention_backward(a["q"], a.pop("q"), a.pop("k"), a.pop("v"), a.pop("out"), torch.zeros(4, 2, 6), a.pop("heads"), **a)


@pytest.mark.parametrize("scale", [1e39, 3e38, float("inf"), 1e-46, 1e-38, -1.0])
def test_refuses_a_scale_outside_fp32(scale):
    """A scale that fp32 turns into infinity, zero or a value whose log2(e)-fold is infinite would give NaN or the mean of the values."""
    from mimo_amd import lib, ops
    with pytest.raises(lib.MimoHipError, match="2\\^126"):
        ops.cross_attention(**_host(scale=scale))
    p = lib.CrossAttentionParams(4, 2, 6, 5, 2, 2, 32, scale, 384, 64, 320, 64, 320, 64)
    L = lib.load()
    assert L.mimo_cross_attention(lib.F16, 4096, 4096, 4096, 4096, None, ctypes.byref(p), None, 0, None) == -1
    assert L.mimo_cross_attention_workspace(ctypes.byref(p)) == L.mimo_cross_attention_backward_workspace(ctypes.byref(p)) == 0


def test_c_entry_refuses_what_it_cannot_run():
    """The C-ABI itself (no device is touched: every one of these returns before a launch)."""
    from mimo_amd import lib
    L = lib.load()
    ok = dict(B=4, Be=2, Nq=6, Nk=5, heads=2, kv_heads=2, d=32, scale=0.1, q_batch=384, q_row=64, k_batch=320, k_row=64, v_batch=320,
              v_row=64, dout_batch=384, dout_row=64)

    def params(**kw):
        p = lib.CrossAttentionParams()
        for n, x in dict(ok, **kw).items():
            setattr(p, n, x)
        return p

    def fwd(p, q=4096, out=4096, ws=None, nb=0, dtype=lib.F16):
        return L.mimo_cross_attention(dtype, q, 4096, 4096, out, None, ctypes.byref(p), ws, nb, None)

    def bwd(p, dout=4096, ws=4096, nb=1 << 30):
        return L.mimo_cross_attention_backward(lib.F16, dout, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096, ctypes.byref(p), ws, nb, None)

    bad = [dict(B=3), dict(B=0), dict(Be=0), dict(Nq=0), dict(Nk=-1), dict(heads=3), dict(kv_heads=0), dict(d=0), dict(d=36), dict(d=168),
           dict(scale=0.0), dict(scale=-1.0), dict(q_row=65), dict(k_batch=4), dict(v_row=12), dict(Nq=1 << 30), dict(Be=1 << 16, B=1 << 16)]
    for kw in bad:
        assert fwd(params(**kw)) == -1 and bwd(params(**kw)) == -1, kw
        assert L.mimo_cross_attention_workspace(ctypes.byref(params(**kw))) == 0
    assert fwd(params(), q=None) == -1 and fwd(params(), out=None) == -1 and fwd(params(), q=4104) == -1
    assert fwd(params(), dtype=7) == -2
    assert bwd(params(), dout=None) == -1 and bwd(params(), ws=None) == -1 and bwd(params(), nb=16) == -1
    assert bwd(params(dout_row=4)) == -1
    long = params(B=2, Nq=1, Nk=100000)   # cut into parts: the workspace is needed and its size is checked
    need = L.mimo_cross_attention_workspace(ctypes.byref(long))
    assert need > 0
    assert fwd(long) == -1 and fwd(long, ws=4096, nb=need - 4) == -1 and fwd(long, ws=4100, nb=need) == -1
    assert L.mimo_cross_attention(lib.F16, 4096, 4096, 4096, 4096, None, None, None, 0, None) == -1
    # without keys: nothing to split, and the backward's scratch is delta alone
    assert L.mimo_cross_attention_workspace(ctypes.byref(params(Nk=0))) == 0
    assert L.mimo_cross_attention_backward_workspace(ctypes.byref(params(Nk=0))) == 4 * 4 * 6 * 2
