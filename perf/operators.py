"""Cross attention to an encoder's states and low-rank adapters beside a shared projection: the cases that are timed, their
plain forms and their definitions in 64 bits.

Two operators, each forward and with its gradients:

  attention   out = softmax(scale q k^T + mask) v for queries that belong to B images and keys / values of Be encoder rows
              (B % Be == 0: the frames of a clip share their text or image embedding), any two lengths, key heads shared by
              groups of query heads, keys cut off by a length per encoder row or a mask; a row without a key gives zeros.
  adapters    out = a w^T + bias + residual + s[i] (a down[i]^T) up[i]^T, i = the adapter of the row's request (or none).

Shapes are token-major as in the rest of the package: [images, tokens, heads * head width], [rows, channels].
"""
import math
import random
from contextlib import nullcontext

import torch

own = False

DEV = "cuda"
HALF = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases --------------------------------------------------------------------------------------------------------
def _att(name, train, dtype, B, Nq, heads, d, Be, Nk, keys="full", kv_heads=None):
    return dict(name=name, op="attention", train=train, dtype=dtype, B=B, Nq=Nq, heads=heads, kv_heads=kv_heads or heads, d=d, Be=Be,
                Nk=Nk, keys=keys)


def _ada(name, train, dtype, M, K, N, S, r, rows="groups", requests=1, out="half"):
    return dict(name=name, op="adapters", train=train, dtype=dtype, M=M, K=K, N=N, S=S, r=r, rows=rows, requests=requests, out=out)


def listed():
    return [
        # the 8 x 8 level of a small preview (4 frames, both halves of a guided batch) on 16 image tokens: a launch and little else
        _att("attention 8x8 preview", False, "fp16", 8, 64, 8, 160, 2, 16),
        # the 64 x 64 level of a 24-frame clip, guided, 77 token states of unequal lengths: the largest ordinary call
        _att("attention 64x64 clip", False, "fp16", 48, 4096, 8, 40, 2, 77, "lengths"),
        # the 32 x 32 level on all 257 states of the image encoder, some masked out
        _att("attention 32x32 image states", False, "bf16", 48, 1024, 8, 80, 2, 257, "mask"),
        # one query token for each of 64 requests over its own long encoder memory, key heads shared by eight query heads
        _att("attention single tokens", False, "bf16", 64, 1, 16, 64, 64, 4097, "lengths", kv_heads=2),
        # fine-tuning the conditioning at the 64 x 64 level: forward and gradients of two 8-frame clips
        _att("attention 64x64 training", True, "fp16", 16, 4096, 8, 40, 2, 77, "lengths"),
        # the same at the 16 x 16 level over image states, a frame size that is no multiple of a tile
        _att("attention 15x17 training", True, "bf16", 24, 255, 8, 160, 3, 257, "mask"),
        # eight requests, one row each, of different adapters: one token or one pooled embedding per request
        _ada("adapters single rows", False, "bf16", 8, 1280, 1280, 8, 16, "tokens", 8),
        # a guided clip at the 64 x 64 level, one adapter for each half
        _ada("adapters 64x64 clip", False, "fp16", 196608, 320, 320, 2, 16, "groups", 2),
        # sixteen requests of unequal lengths through a 1280-wide projection into the fp32 residual stream
        _ada("adapters ragged requests", False, "bf16", 12321, 1280, 1280, 16, 64, "ragged", 16, "f32"),
        # keys and values of an encoder's states: few rows, another width on each side
        _ada("adapters encoder states", False, "fp16", 514, 768, 640, 2, 8, "groups", 2),
        # training one adapter at the 32 x 32 level
        _ada("adapters 32x32 training", True, "fp16", 49152, 640, 640, 1, 32, "groups", 1),
        # training several at once on a ragged batch
        _ada("adapters ragged training", True, "bf16", 5003, 1280, 640, 7, 24, "ragged", 9),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    train = rng.random() < 0.4
    if rng.random() < 0.5:
        d = rng.choice([8, 24, 40, 64, 72, 80, 96, 128, 160])
        kvh = rng.choice([1, 2, 4, 8])
        heads = kvh * rng.choice([1, 1, 1, 2, 8] if kvh < 4 else [1, 1, 2])
        Be = _spread(rng, 1, 16)
        B = Be * _spread(rng, 1, 24)
        if rng.random() < 0.25:  # few queries over a long memory
            Nq, Nk = _spread(rng, 1, 16), _spread(rng, 64, 20000)
        else:
            # (the scores of a single key have no gradient: dq and dk would be nothing but rounding)
            Nq, Nk = _spread(rng, 16, 4096), _spread(rng, 8 if train else 1, 1024)
        # at most the scores and the bytes of the largest listed cases
        most, each = (4.6e7, 8) if train else (1.2e8, 4)
        while B * heads * Nq * Nk > most or each * d * (B * Nq * heads + Be * Nk * kvh) > 2.5e8 or B * heads * Nk * d > 2.6e8:
            if Nq > 16 and Nq * 4 > Nk:
                Nq = (Nq + 1) // 2
            elif B > Be:
                B = Be * max(1, B // Be // 2)
            elif Be > 1:
                B = Be = Be // 2
            else:
                Nq, Nk = (Nq + 1) // 2, (Nk + 1) // 2
        c = _att("", train, dtype, B, Nq, heads, d, Be, Nk, rng.choice(["full", "lengths", "lengths", "mask"]), kvh)
    else:
        K, N = (8 * _spread(rng, 5, 160) for _ in range(2))
        M = _spread(rng, 1, 200000)
        out = "half" if train else rng.choice(["half", "half", "f32"])
        while M * max(K, N) > (3.1e7 if train else 6.2e7 if out == "half" else 2.5e7) or M * K * N > 2e10:
            M = (M + 1) // 2
        rows = rng.choice(["tokens", "groups", "ragged"]) if M <= 512 else rng.choice(["groups", "ragged"])
        requests = M if rows == "tokens" else min(M, _spread(rng, 1, 40))
        S = _spread(rng, 1, 24)
        r = 8 * _spread(rng, 1, 16)
        while S * r > 1024:
            S = (S + 1) // 2
        c = _ada("", train, dtype, M, K, N, S, r, rows, requests, out)
    del c["name"]
    return c


# ---- what depends on the case alone: lengths, masks, which request has which adapter -----------------------------------------
def _rng(c):
    return random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))


def _lengths(c):
    """Valid keys of each encoder row: from a third of them to all; where there are more than two rows, one has none."""
    if c["keys"] != "lengths":
        return None
    rng = _rng(c)
    n = [rng.randint((c["Nk"] + 2) // 3, c["Nk"]) for _ in range(c["Be"])]
    n[0] = c["Nk"]
    if c["Be"] > 2:
        n[rng.randrange(1, c["Be"])] = 0
    return n


def _mask(c):
    """[Be][Nk] truth values, three in four keys attended; where there are more than two rows, one is empty."""
    if c["keys"] != "mask":
        return None
    g = torch.Generator().manual_seed(_rng(c).randrange(1 << 30))
    m = torch.rand((c["Be"], c["Nk"]), generator=g) < 0.75
    m[0, 0] = True
    if c["Be"] > 2:
        m[1 + _rng(c).randrange(c["Be"] - 1)] = False
    return m


def _valid(c):
    """Valid keys of each encoder row, as a list."""
    if c["keys"] == "lengths":
        return _lengths(c)
    if c["keys"] == "mask":
        return [int(x) for x in _mask(c).sum(1)]
    return [c["Nk"]] * c["Be"]


def _index(c):
    """(adapter of each request's rows as a list, rows that share an entry): -1 where a request has none."""
    rng = _rng(c)
    n, S = c["requests"], c["S"]
    who = [i % S for i in range(n)]
    if n > 1:
        rng.shuffle(who)
    if n > 3:
        who[rng.randrange(n)] = -1
    if c["rows"] == "tokens":
        return who, 1
    if c["rows"] == "groups":
        per = (c["M"] + n - 1) // n
        return who[: (c["M"] + per - 1) // per], per
    cuts = sorted(rng.sample(range(1, c["M"]), n - 1)) if n > 1 else []
    each = [b - a for a, b in zip([0] + cuts, cuts + [c["M"]])]
    return [w for w, k in zip(who, each) for _ in range(k)], 1


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = HALF[c["dtype"]]

    def rnd(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)

    if c["op"] == "attention":
        B, Be, C, Ck = c["B"], c["Be"], c["heads"] * c["d"], c["kv_heads"] * c["d"]
        kv = rnd(Be, c["Nk"], 2 * Ck)  # one projection of the encoder's states gives both: k and v are views of it
        n, m = _lengths(c), _mask(c)
        s = dict(c, q=rnd(B, c["Nq"], C), k=kv[..., :Ck], v=kv[..., Ck:], kv_len=None, mask=None)
        if n is not None:
            s["kv_len"] = torch.tensor(n, dtype=torch.int32, device=DEV)
            kv.masked_fill_((torch.arange(c["Nk"], device=DEV)[None] >= s["kv_len"][:, None])[..., None], float("nan"))  # padding holds anything
        if m is not None:
            s["mask"] = m.to(DEV)
        if c["train"]:
            s["dout"] = rnd(B, c["Nq"], C)
        return s
    M, K, N, S, r = (c[x] for x in ("M", "K", "N", "S", "r"))
    who, per = _index(c)
    s = dict(c, a=rnd(M, K), w=rnd(N, K, scale=K ** -0.5), down=rnd(S, r, K, scale=K ** -0.5), up=rnd(S, N, r, scale=0.5 * r ** -0.5),
             index=torch.tensor(who, dtype=torch.int32, device=DEV), per=per, scale=rnd(S, dtype=torch.float32).abs() + 0.5,
             bias=rnd(N, dtype=torch.float32), residual=rnd(M, N, dtype=torch.float32) if c["out"] == "f32" else None)
    if c["train"]:
        s["dout"] = rnd(M, N)
        s["w_t"] = s["w"].t().contiguous()  # the frozen weight, laid out once for the gradient of the input
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    with torch.no_grad():
        if own:
            return _own(state)
        return _plain_attention(state) if state["op"] == "attention" else _plain_adapters(state)


def _own(s):
    from mimo_amd import ops
    if s["op"] == "attention":
        kw = dict(kv_heads=s["kv_heads"], kv_len=s["kv_len"], mask=s["mask"])
        if not s["train"]:
            return ops.cross_attention(s["q"], s["k"], s["v"], s["heads"], **kw)
        out, lse = ops.cross_attention(s["q"], s["k"], s["v"], s["heads"], want_lse=True, **kw)
        dq, dk, dv = ops.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, s["heads"], **kw)
        return dict(out=out, dq=dq, dk=dk, dv=dv)
    kw = dict(rows_per_index=s["per"], scale=s["scale"])
    if not s["train"]:
        return ops.adapter_gemm(s["a"], s["w"], s["down"], s["up"], s["index"], bias=s["bias"], residual=s["residual"],
                                out_f32=s["out"] == "f32", **kw)
    out, low = ops.adapter_gemm(s["a"], s["w"], s["down"], s["up"], s["index"], bias=s["bias"], want_low=True, **kw)
    da, ddown, dup = ops.adapter_gemm_backward(s["dout"], s["a"], s["w_t"], s["down"], s["up"], s["index"], low, **kw)
    return dict(out=out, da=da, ddown=ddown, dup=dup)


def _heads(x, n):
    """[images, tokens, n * d] -> fp32 [images, n, tokens, d]."""
    return x.float().unflatten(2, (n, -1)).transpose(1, 2).contiguous()


def _plain_attention(s):
    B, Be, H, G = s["B"], s["Be"], s["heads"], s["kv_heads"]
    rep = B // Be
    scale = s["d"] ** -0.5
    keep = torch.ones((Be, s["Nk"]), dtype=torch.bool, device=s["q"].device)
    if s["kv_len"] is not None:
        keep = torch.arange(s["Nk"], device=keep.device)[None] < s["kv_len"][:, None]
    if s["mask"] is not None:
        keep = s["mask"]
    q = _heads(s["q"], H)
    k = _heads(s["k"].masked_fill(~keep[..., None], 0), G).repeat_interleave(rep, 0).repeat_interleave(H // G, 1)
    v = _heads(s["v"].masked_fill(~keep[..., None], 0), G).repeat_interleave(rep, 0).repeat_interleave(H // G, 1)
    row = keep.repeat_interleave(rep, 0)[:, None, None, :]
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).masked_fill_(~row, float("-inf"))
    top = p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)  # a row without a key: exp(-inf - lowest) = 0
    p = p.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny))

    def tokens(x):
        return x.transpose(1, 2).flatten(2).to(s["q"].dtype)

    o = torch.matmul(p, v)
    if not s["train"]:
        return tokens(o)
    do = _heads(s["dout"], H)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)

    def shared(x):  # the gradient of what `rep` images and H / G query heads share is their sum
        return tokens(x.unflatten(0, (Be, rep)).sum(1).unflatten(1, (G, H // G)).sum(2))

    return dict(out=tokens(o), dq=tokens(torch.matmul(ds, k)), dk=shared(torch.matmul(ds.transpose(2, 3).contiguous(), q)),
                dv=shared(torch.matmul(p.transpose(2, 3).contiguous(), do)))


def _plain_adapters(s):
    S, r, N, K = s["S"], s["r"], s["N"], s["K"]
    a, w, down, up = (s[x].float() for x in ("a", "w", "down", "up"))
    who = s["index"].repeat_interleave(s["per"])[: s["M"]]
    pick = (who[:, None] == torch.arange(S, device=who.device)[None]).float() * s["scale"][None]  # [M, S]: s[i] at the row's adapter
    flat_down, flat_up = down.reshape(S * r, K), up.permute(0, 2, 1).reshape(S * r, N)
    low = ((a @ flat_down.t()).unflatten(1, (S, r)) * pick[..., None]).flatten(1)
    out = a @ w.t() + s["bias"] + low @ flat_up
    if s["residual"] is not None:
        out = out + s["residual"]
    out = out if s["out"] == "f32" else out.to(s["a"].dtype)
    if not s["train"]:
        return out
    dy = s["dout"].float()
    dlow = ((dy @ flat_up.t()).unflatten(1, (S, r)) * pick[..., None]).flatten(1)
    da = dy @ w + dlow @ flat_down
    return dict(out=out, da=da.to(s["a"].dtype), ddown=(dlow.t() @ a).reshape(S, r, K),
                dup=(low.t() @ dy).reshape(S, r, N).transpose(1, 2).contiguous())


# ---- the work that cannot be left out ------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "attention":
        rep, C, Ck = c["B"] // c["Be"], c["heads"] * c["d"], c["kv_heads"] * c["d"]
        pairs = sum(_valid(c)) * rep * c["Nq"]
        q, kv = 2 * c["B"] * c["Nq"] * C, 2 * 2 * sum(_valid(c)) * Ck
        if not c["train"]:  # q, k, v read; out written
            return dict(bytes=2 * q + kv, flops=4 * pairs * C)
        return dict(bytes=4 * q + kv + 2 * 2 * c["Be"] * c["Nk"] * Ck, flops=12 * pairs * C)  # + dout read, dq, dk, dv written
    M, K, N, S, r = (c[x] for x in ("M", "K", "N", "S", "r"))
    who, per = _index(c)
    used = len({w for w in who if w >= 0})
    rows = sum(per if i < len(who) - 1 else M - per * (len(who) - 1) for i, w in enumerate(who) if w >= 0)
    weights = 2 * N * K + 2 * used * r * (N + K)
    out = (4 + 4) * M * N if c["out"] == "f32" else 2 * M * N
    fwd = dict(bytes=2 * M * K + weights + out, flops=2 * M * N * K + 2 * rows * r * (N + K))
    if not c["train"]:
        return fwd
    return dict(bytes=fwd["bytes"] + 2 * M * N + 2 * M * K + 4 * S * r * (N + K),
                flops=fwd["flops"] + 2 * M * N * K + 2 * rows * r * (N + K) + 2 * rows * r * (N + K))


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.enable_grad() if c["train"] else nullcontext():
        return _exact_attention(c, s) if c["op"] == "attention" else _exact_adapters(c, s)


def _exact_attention(c, s):
    rep, H, G, d = c["B"] // c["Be"], c["heads"], c["kv_heads"], c["d"]
    n, m = _lengths(c), _mask(c)
    res = dict(out=torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV))
    if c["train"]:
        res.update(dq=torch.zeros_like(res["out"]), dk=torch.zeros(s["k"].shape, dtype=torch.float64, device=DEV),
                   dv=torch.zeros(s["v"].shape, dtype=torch.float64, device=DEV))
    for e in range(c["Be"]):
        at = torch.arange(n[e] if n is not None else c["Nk"], device=DEV) if m is None else m[e].nonzero()[:, 0].to(DEV)
        if at.numel() == 0:
            continue
        for h in range(G):  # the keys that count, and the queries (images, tokens, query heads of this key head) that see them
            k, v = (s[x][e, at, h * d:(h + 1) * d].double().requires_grad_(c["train"]) for x in "kv")
            for i in range(e * rep, (e + 1) * rep):
                cols = slice(h * (H // G) * d, (h + 1) * (H // G) * d)
                q = s["q"][i, :, cols].double().reshape(-1, d).requires_grad_(c["train"])
                o = torch.softmax(q @ k.t() / math.sqrt(d), -1) @ v
                res["out"][i, :, cols] = o.detach().reshape(c["Nq"], -1)
                if c["train"]:
                    o.backward(s["dout"][i, :, cols].double().reshape(-1, d))
                    res["dq"][i, :, cols] = q.grad.reshape(c["Nq"], -1)
            if c["train"]:
                res["dk"][e, at, h * d:(h + 1) * d] = k.grad
                res["dv"][e, at, h * d:(h + 1) * d] = v.grad
    return res if c["train"] else res["out"]


def _exact_adapters(c, s):
    who, per = _index(c)
    who = torch.tensor(who, device=DEV).repeat_interleave(per)[: c["M"]]
    w = s["w"].double()
    out = torch.empty((c["M"], c["N"]), dtype=torch.float64, device=DEV)
    da = torch.empty((c["M"], c["K"]), dtype=torch.float64, device=DEV) if c["train"] else None
    down, up = (s[x].double().requires_grad_(c["train"]) for x in ("down", "up"))
    for i in range(-1, c["S"]):
        at = (who == i).nonzero()[:, 0]
        a = s["a"][at].double().requires_grad_(c["train"])
        y = torch.nn.functional.linear(a, w, s["bias"].double())
        if i >= 0:
            y = y + float(s["scale"][i]) * ((a @ down[i].t()) @ up[i].t())
        out[at] = y.detach() if s["residual"] is None else y.detach() + s["residual"][at].double()
        if c["train"]:
            y.backward(s["dout"][at].double())
            da[at] = a.grad
    return dict(out=out, da=da, ddown=down.grad, dup=up.grad) if c["train"] else out
