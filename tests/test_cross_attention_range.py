"""Gradients of the cross attention far from order one: an unscaled mean loss (small dO), a scaled loss (large dO), values of other
sizes, keys that are hardly looked at.  Relative L2 against the formulas in 64 bits.

What may be left of dq, dk and dv are the roundings to the operand type that the kernels make, each relative to the value that is
rounded WHATEVER its size: dS (dq and dk), P (dv), the stored output (through delta) and the result.  A rounding is uniform within
half a step u = eps / 2, mantissas spread evenly in their logarithm: 0.425 u of the value in the mean square, independent of each
other; 15 % for the sample.  The stored output o = sum_k P v carries two of them, its own and P's: with e_k = P's relative error,
delta = sum_c dO_c o_c is off by sum_c dO_c sum_k e_k P_k v_kc = sum_k e_k P_k dP_k from the second.  Absolute are only the operands'
own formats: half of the smallest step (2^-25 in fp16) on the result and on the stored output."""
import pytest
import torch

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch.device("cuda:0")


def operands(case, dtype):
    """CPU tensors (q, k, v, dout) of a case."""
    B, Be, Nq, Nk, heads, kvh, d, sizes = case
    g = torch.Generator().manual_seed(Nq + Nk + d)
    shapes = ((B, Nq, heads * d), (Be, Nk, kvh * d), (Be, Nk, kvh * d), (B, Nq, heads * d))
    return [(torch.randn(s, generator=g) * x).to(dtype) for s, x in zip(shapes, sizes)]


def expected(case, q, k, v, dout):
    """Values in 64 bits and, for each, the error in the mean square that the roundings leave (as the norm over all elements)."""
    B, Be, Nq, Nk, heads, kvh, d, _ = case
    rep, hg, c = B // Be, heads // kvh, d ** -0.5
    r, tiny = 0.425 * torch.finfo(q.dtype).eps / 2, 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    rows = lambda x: x.double().reshape(Be, rep, Nq, kvh, hg, d).permute(0, 3, 1, 2, 4, 5).reshape(Be, kvh, -1, d)
    back = lambda x: x.reshape(Be, kvh, rep, Nq, hg, d).permute(0, 2, 3, 1, 4, 5).reshape(B, Nq, heads * d)
    keys = lambda x: x.double().reshape(Be, Nk, kvh, d).transpose(1, 2)
    Q, G, K, V = rows(q), rows(dout), keys(k), keys(v)
    P = (Q @ K.transpose(2, 3) * c).softmax(-1)
    O, dP = P @ V, G @ V.transpose(2, 3)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    delta2 = ((G * O).square() * r * r + G.square() * tiny * tiny).sum(-1, keepdim=True) + (P * dP).square().sum(-1, keepdim=True) * r * r
    if Nk <= 32:   # delta = sum_k P dP there
        delta2 = torch.zeros_like(delta2)
    val = dict(dq=c * dS @ K, dk=c * dS.transpose(2, 3) @ Q, dv=P.transpose(2, 3) @ G)
    err2 = dict(dq=c * c * ((dS.square() @ K.square()) * r * r + delta2 * (P @ K).square()),
                dk=c * c * ((dS.square().transpose(2, 3) @ Q.square()) * r * r + P.square().transpose(2, 3) @ (delta2 * Q.square())),
                dv=(P.square().transpose(2, 3) @ G.square()) * r * r)
    left = {n: float((err2[n].sum() + r * r * val[n].square().sum() + tiny * tiny * val[n].numel()).sqrt()) for n in val}
    return dict(dq=back(val["dq"]), dk=val["dk"].transpose(1, 2).flatten(2), dv=val["dv"].transpose(1, 2).flatten(2)), left


#   B  Be  Nq    Nk  heads kvh d   sizes of q, k, v, dO
CASES = [
    (1, 1, 4096, 77, 2, 2, 40, (1, 1, 1, 1e-4)),       # a mean loss over a level's rows
    (2, 1, 512, 1024, 2, 2, 40, (1, 1, 1, 1e-3)),      # many keys: P itself is small
    (2, 2, 700, 300, 2, 2, 160, (1, 1, 1, 1e-3)),      # streamed, waves that share a key tile
    (4, 2, 300, 257, 4, 2, 80, (1, 1, 1e-3, 0.1)),     # small values
    (2, 2, 600, 128, 2, 2, 16, (1, 1, 1, 1e-3)),       # narrow heads
    (64, 4, 1, 3000, 8, 1, 64, (1, 1, 1, 1e-2)),       # single tokens over a long memory
    (2, 2, 100, 20, 2, 2, 96, (1, 1, 1, 1e-4)),        # few keys
    (1, 1, 64, 100, 2, 2, 160, (1.5, 1.5, 1, 1e4)),    # a scaled loss on a peaked softmax: dS passes 65504, dq does not
    (2, 2, 16, 33, 2, 2, 64, (1.5, 1.5, 8, 2e3)),
    (8, 2, 20, 300, 2, 2, 160, (1.7, 1.7, 16, 6e2)),
    (2, 2, 32, 40, 2, 2, 24, (1, 1, 60, 5e2)),
]


@pytest.mark.parametrize("case", CASES)
def test_cases_reach_where_the_16_bit_range_ends(case):
    """dS passes the largest fp16 or lies mostly below its normal range, while every gradient fits."""
    q, k, v, dout = operands(case, torch.float16)
    val, _ = expected(case, q, k, v, dout)
    assert all(float(x.abs().max()) < 65000 for x in val.values())
    B, Be, Nq, Nk, heads, kvh, d, sizes = case
    split = lambda x, n, rep: x.double().reshape(x.shape[0], -1, n, d).transpose(1, 2).repeat_interleave(rep, 0)
    Q, G = split(q, heads, 1), split(dout, heads, 1)
    K, V = (split(x, kvh, B // Be).repeat_interleave(heads // kvh, 1) for x in (k, v))
    P, dP = (Q @ K.transpose(2, 3) * d ** -0.5).softmax(-1), G @ V.transpose(2, 3)
    dS = (P * (dP - (P * dP).sum(-1, keepdim=True))).abs()
    assert float(dS.max()) > 65504 if sizes[3] > 1 else float((dS < 2.0 ** -14).double().mean()) > 0.5


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_gradients_of_any_size(dev, dtype, case):
    from mimo_amd import ops
    heads, kvh = case[4], case[5]
    q, k, v, dout = (x.to(dev) for x in operands(case, dtype))
    out, lse = ops.cross_attention(q, k, v, heads, kv_heads=kvh, want_lse=True)
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kvh)
    val, left = expected(case, q, k, v, dout)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert torch.isfinite(got).all(), name
        off = float((got.double() - val[name]).norm())
        assert off <= 1.15 * left[name], (name, off, left[name], float(val[name].norm()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 1, 64, 60000, 2, 2, 40, (1, 1, 1, 1)), (8, 1, 2, 40000, 2, 1, 160, (1, 1, 1, 1))])
def test_value_gradient_of_keys_that_are_hardly_seen(dev, dtype, case):
    """Among tens of thousands of keys P is below the normal range of fp16, dv = P^T dO is not."""
    from mimo_amd import ops
    heads, kvh = case[4], case[5]
    q, k, v, dout = (x.to(dev) for x in operands(case, dtype))
    out, lse = ops.cross_attention(q, k, v, heads, kv_heads=kvh, want_lse=True)
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kvh)
    val, left = expected(case, q, k, v, dout)
    for name, got in zip(("dq", "dk", "dv"), grads):
        off = float((got.double() - val[name]).norm())
        assert off <= 1.15 * left[name], (name, off, left[name], float(val[name].norm()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Nk,d,heads", [(70, 40, 1), (64, 160, 1), (33, 16, 2), (300, 160, 1), (900, 128, 1), (1500, 24, 1), (257, 80, 1)])
def test_one_large_value_anywhere(dev, dtype, Nk, d, heads):
    """dS is held relative to a bound that contains the largest |v|: one value of 6e4 among others of 1e-3, at another key and channel in
    each of 192 encoder rows, so that every lane and wave that looks for it has it once.  Missed, dS would be infinite.  A key that
    does not count may hold anything."""
    from mimo_amd import ops
    E, Nq = 192, 33
    q, k, v, dout = (x.to(dev) for x in operands((E, E, Nq, Nk, heads, heads, d, (1, 1, 1e-3, 1e-2)), dtype))
    at = torch.randperm((Nk - 1) * heads * d, generator=torch.Generator().manual_seed(3))[:E].to(dev)
    v.view(E, -1)[torch.arange(E, device=dev), at] = 6e4
    v[:, -1], k[:, -1] = 65504.0, float("nan")
    kv_len = torch.full((E,), Nk - 1, dtype=torch.int32, device=dev)
    out, lse = ops.cross_attention(q, k, v, heads, kv_len=kv_len, want_lse=True)
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_len=kv_len)
    val, left = expected((E, E, Nq, Nk - 1, heads, heads, d, None), q, k[:, :-1], v[:, :-1], dout)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert torch.isfinite(got).all(), name
        got = got if name == "dq" else got[:, :-1]
        off = float((got.double() - val[name]).norm())
        assert off <= 1.15 * left[name], (name, off, left[name], float(val[name].norm()))
