"""Encoder states of several tokens: the UNets conditioned on them against the CPU oracle, and a cross-attention layer whose four
projections carry adapters (adapter_gemm around cross_attention), forward and backward, against the formulas in 64 bits."""
import pytest
import torch

from conftest import rel_l2
from helpers import build_pair_unets

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
# the whole-model bars of the same half-width models with one token
TOL_UNET = {torch.float16: 3e-3, torch.bfloat16: 3e-2}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch.device("cuda:0")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hw,F,L", [(16, 3, 77), (13, 2, 5)])
def test_unets_on_several_tokens(dev, dtype, hw, F, L):
    """The denoising UNet (frames share their row's tokens) and the reference UNet, without and with a mask: a masked row is the
    oracle's on the tokens that are left."""
    o3, o2, p3, p2 = build_pair_unets(dtype, dev)
    g = torch.Generator().manual_seed(16)
    ehs = torch.randn(2, L, 768, generator=g)
    x, pose = torch.randn(2, 8, F, hw, hw, generator=g), torch.randn(2, 160, F, hw, hw, generator=g)
    lat = torch.randn(2, 4, hw, hw, generator=g)
    mask = torch.rand(2, L, generator=g) < 0.5
    mask[:, 1] = True
    t = 749
    with torch.no_grad():
        ref3, ref2 = o3(x, torch.tensor(t), ehs, pose_cond_fea=pose), o2(lat, torch.zeros(()), ehs)
        masked3 = torch.cat([o3(x[i:i + 1], torch.tensor(t), ehs[i:i + 1, mask[i]], pose_cond_fea=pose[i:i + 1]) for i in range(2)])
    out3 = p3(x.to(dev), t, ehs.to(dev), pose_cond_fea=pose.to(dev)).sample.cpu()
    out2 = p2(lat.to(dev), 0, ehs.to(dev)).sample.cpu()
    assert rel_l2(out3, ref3) < TOL_UNET[dtype] and rel_l2(out2, ref2) < TOL_UNET[dtype]
    got = [p3(x.to(dev), t, ehs.to(dev), pose_cond_fea=pose.to(dev), encoder_attention_mask=m.to(dev)).sample.cpu() for m in (mask, mask.long())]
    assert rel_l2(got[0], masked3) < TOL_UNET[dtype] and torch.equal(got[0], got[1])
    assert rel_l2(got[0], ref3) > rel_l2(got[0], masked3)
    # tokens that the mask drops have no say
    other = torch.where(mask[..., None], ehs, torch.full_like(ehs, float("nan")))
    assert torch.equal(p3(x.to(dev), t, other.to(dev), pose_cond_fea=pose.to(dev), encoder_attention_mask=mask.to(dev)).sample.cpu(), got[0])


@gpu
def test_one_token_with_a_mask_is_the_collapsed_path(dev):
    """One token that counts: the attention gives its value, which is what the collapsed form folds into one matrix; one that does
    not: only the output projection's bias is added, as if the weights of the values were zero."""
    _, _, p3, _ = build_pair_unets(torch.float16, dev)
    g = torch.Generator().manual_seed(17)
    ehs, x = torch.randn(1, 1, 768, generator=g).to(dev), torch.randn(1, 8, 2, 8, 8, generator=g).to(dev)
    plain = p3(x, 400, ehs).sample
    kept = p3(x, 400, ehs, encoder_attention_mask=torch.ones(1, 1, dtype=torch.bool, device=dev)).sample
    dropped = p3(x, 400, ehs, encoder_attention_mask=torch.zeros(1, 1, dtype=torch.bool, device=dev)).sample
    assert torch.equal(p3(x, 400, ehs).sample, plain)  # the packed copies of the two paths live side by side
    nothing = p3(x, 400, torch.zeros_like(ehs)).sample
    tol = TOL_UNET[torch.float16]
    assert rel_l2(kept, plain) < tol and rel_l2(dropped, nothing) < tol and rel_l2(dropped, plain) > tol


def test_refusals_of_several_tokens():
    from mimo_amd.modules import Ctx
    _, _, p3, p2 = build_pair_unets(torch.float16, torch.device("cpu"))
    many, one = torch.randn(2, 7, 768), torch.randn(2, 1, 768)
    keep = torch.ones(2, 7, dtype=torch.bool)
    with pytest.raises(ValueError, match="one token per row"):
        p3.clip_tables([749], many, 2)
    for kw in (dict(ehs=many, ehs_mask=None), dict(ehs=one, ehs_mask=keep[:, :1])):
        p2.precision = "split"
        with pytest.raises(ValueError, match="precision"):
            p2.run_tokens(None, 0, b=2, F=1, **kw)
        p2.precision = "half"
        with pytest.raises(ValueError, match="precision"):
            p2.run_tokens(None, 0, b=2, F=1, temb=torch.zeros(2, 1), attn2=torch.zeros(2, 1), **kw)
    for ehs, mask in ((many[:1], None), (torch.randn(2, 7, 64), None), (many[:, :0], keep[:, :0]), (many, keep[:, :6]), (many, keep[0]),
                      (many, keep.float())):
        with pytest.raises(ValueError, match="encoder_"):
            p3._tokens(Ctx(torch.float16, 2, 1), ehs, mask)
    ctx = Ctx(torch.float16, 2, 1)
    p3._tokens(ctx, one, None)
    assert ctx.tokens is None
    p3._tokens(ctx, many, keep)
    assert ctx.tokens.dtype == torch.float16 and ctx.tokens_mask.dtype == torch.uint8


def test_refusal_of_several_tokens_with_a_split_module():
    """A single spatial transformer on split operands takes the collapsed form only: refused before anything has run (no bank is
    written).  One token runs as before, and so does a split module of another kind."""
    from mimo_amd.modules import SpatialTransformer
    _, _, p3, p2 = build_pair_unets(torch.float16, torch.device("cpu"))
    many, one = torch.randn(2, 7, 768), torch.randn(2, 1, 768)
    keep = torch.ones(2, 7, dtype=torch.bool)
    for u in (p3, p2):
        all_of_it = [m for m in u.modules() if isinstance(m, SpatialTransformer)]
        assert len(all_of_it) == 16
        for m in all_of_it:
            m.precision = "split"
            for kw in (dict(ehs=many), dict(ehs=many, ehs_mask=keep), dict(ehs=one, ehs_mask=keep[:, :1])):
                with pytest.raises(ValueError, match="spatial transformers"):
                    u.run_tokens(None, 0, b=2, F=1, **kw)
            del m.precision
        u.up_blocks[-1].resnets[-1].precision = "split"
        with pytest.raises(ValueError, match="encoder_"):   # (past the refusal: the shape is looked at next)
            u.run_tokens(None, 0, many[:1], 2, 1)


def test_packed_projections_follow_the_weights():
    _, _, p3, _ = build_pair_unets(torch.float16, torch.device("cpu"))
    blk = p3.spatial_blocks()[0]
    first = blk.packed_tokens(torch.float16)
    assert blk.packed_tokens(torch.float16) is first
    with torch.no_grad():
        blk.attn2.to_q.weight.add_(1.0)
    p3.load_state_dict(p3.state_dict())
    assert torch.equal(blk.packed_tokens(torch.float16)["q"], blk.attn2.to_q.weight.detach().half())
    assert blk.packed_tokens(torch.bfloat16)["q"].dtype == torch.bfloat16


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Be,Nq,Nk,heads,kvh,d,S,r", [(6, 2, 64, 77, 8, 8, 40, 3, 16), (4, 4, 1, 50, 8, 2, 64, 5, 8), (2, 1, 33, 200, 4, 4, 80, 2, 32)])
def test_layer_with_adapters(dev, dtype, B, Be, Nq, Nk, heads, kvh, d, S, r):
    """y = x + o W_o^T .., o = attention(x W_q^T .., e W_k^T .., e W_v^T ..), every projection with the adapter of its image's (its
    encoder row's) request, one request without, one key row masked out.  Relative L2 against autograd in 64 bits.  Each path has at
    most ten roundings to the 16-bit type (projections and their low-rank values, P, the attention's output; as many gradients on the
    way back, the backward recomputing P from rounded operands), each at most u of what it rounds; the softmax at most doubles what
    reaches it through the scores, which are of order one here.  2 x 10 u forward, as much again on the way back."""
    from mimo_amd import ops
    u = torch.finfo(dtype).eps / 2
    C, Ck, Ce = heads * d, kvh * d, 96
    gen = torch.Generator().manual_seed(B * Nk + d)
    rand = lambda *shape, s=1.0: (torch.randn(*shape, generator=gen) * s).to(dtype).to(dev)
    x, e, G = rand(B, Nq, C), rand(Be, Nk, Ce), rand(B, Nq, C)
    dims = dict(q=(C, C), k=(Ck, Ce), v=(Ck, Ce), o=(C, C))
    W = {n: rand(o, i, s=i ** -0.5) for n, (o, i) in dims.items()}
    D = {n: rand(S, r, i, s=i ** -0.5) for n, (o, i) in dims.items()}
    U = {n: rand(S, o, r, s=0.5 * r ** -0.5) for n, (o, i) in dims.items()}
    scale = (torch.rand(S, generator=gen) + 0.5).to(dev)
    image = torch.randint(0, S, (B,), generator=gen, dtype=torch.int32)
    image[-1] = -1
    row = torch.randint(0, S, (Be,), generator=gen, dtype=torch.int32)
    mask = torch.rand(Be, Nk, generator=gen) < 0.7
    mask[0, 0], mask[-1] = True, mask[-1] if Be == 1 else False
    image, row, mask = image.to(dev), row.to(dev), mask.to(dev)

    X, E = x.double().requires_grad_(), e.double().requires_grad_()
    D64 = {n: t.double().requires_grad_() for n, t in D.items()}
    U64 = {n: t.double().requires_grad_() for n, t in U.items()}

    def project(t, n, index):
        y = t @ W[n].double().t()
        parts = [y[i] + (scale[s].double() * (t[i] @ D64[n][s].t()) @ U64[n][s].t() if s >= 0 else 0) for i, s in enumerate(index.tolist())]
        return torch.stack(parts)
    q = project(X, "q", image).view(B, Nq, heads, d).transpose(1, 2)
    k, v = (project(E, n, row).view(Be, Nk, kvh, d).transpose(1, 2).repeat_interleave(B // Be, 0).repeat_interleave(heads // kvh, 1)
            for n in "kv")
    keep = mask.repeat_interleave(B // Be, 0)[:, None, None, :]
    sc = (q @ k.transpose(-1, -2)) * d ** -0.5
    p = torch.where(keep, sc, torch.full_like(sc, -1e30)).softmax(-1) * keep
    o = (p @ v).transpose(1, 2).reshape(B, Nq, C)
    Y = project(o, "o", image) + X
    Y.backward(G.double())

    args = {n: dict(rows_per_index=Nq if n in "qo" else Nk, scale=scale) for n in dims}
    idx = {n: image if n in "qo" else row for n in dims}
    low = {}

    def run(t, n, **kw):
        y, low[n] = ops.adapter_gemm(t, W[n], D[n], U[n], idx[n], want_low=True, **args[n], **kw)
        return y
    xf, ef = x.view(-1, C), e.view(-1, Ce)
    qh, kh, vh = run(xf, "q").view(B, Nq, C), run(ef, "k").view(Be, Nk, Ck), run(ef, "v").view(Be, Nk, Ck)
    oh, lse = ops.cross_attention(qh, kh, vh, heads, kv_heads=kvh, mask=mask, want_lse=True)
    y = run(oh.view(-1, C), "o", residual=xf, out_f32=True)
    assert rel_l2(y.double(), Y.detach().view(-1, C)) < 20 * u

    def back(g, t, n):
        return ops.adapter_gemm_backward(g, t, W[n].t().contiguous(), D[n], U[n], idx[n], low[n], **args[n])
    grads = {}
    do, *grads["o"] = back(G.view(-1, C), oh.view(-1, C), "o")
    dq, dk, dv = ops.cross_attention_backward(do.view(B, Nq, C), qh, kh, vh, oh, lse, heads, kv_heads=kvh, mask=mask)
    dx, *grads["q"] = back(dq.view(-1, C), xf, "q")
    dek, *grads["k"] = back(dk.view(-1, Ck), ef, "k")
    dev_, *grads["v"] = back(dv.view(-1, Ck), ef, "v")
    assert rel_l2(dx.double() + G.view(-1, C).double(), X.grad.view(-1, C)) < 40 * u
    assert rel_l2(dek.double() + dev_.double(), E.grad.view(-1, Ce)) < 40 * u
    for n in dims:
        assert rel_l2(grads[n][0].double(), D64[n].grad) < 40 * u, n
        assert rel_l2(grads[n][1].double(), U64[n].grad) < 40 * u, n
