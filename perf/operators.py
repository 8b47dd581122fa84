"""The operators around the expert block, one call each, as a decoder layer makes them.

kind "norm"    root-mean-square norm behind the residual's addition, its output
               in 16 bits or in e4m3 with a scale per 128 columns:
               ops.add_rms_norm
kind "linear"  8-bit product with a scale per block of 128: ops.linear_fp8
kind "rope"    rotary positions of the new tokens' queries and keys, keys and
               values put into the pages of a cache: ops.rope_cache
kind "attn"    attention of the new tokens over that cache: ops.attn_paged

A batch is `seqs` sequences with 1 to `new` new tokens each behind 0 to `ctx`
cached ones (all of them the most where `ragged` is false).  Head layouts: 32
query and 4 key heads of 128, and 64 and 8 of 64 with a window and sinks, plus
smaller groups.
"""
import math
import random

import torch

own = False

EPS = 1e-6
FP8_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token of a decoding sequence, before the router
        dict(name="norm-1", kind="norm", tokens=1, width=2048, fp8=False, dtype="bf16"),
        # a long prompt's chunk, before the query/key/value product; 22.5 blocks a row
        dict(name="norm-8192-fp8", kind="norm", tokens=8192, width=2880, fp8=True, dtype="bf16"),
        # one token's query/key/value product: the weights' bytes
        dict(name="linear-1", kind="linear", tokens=1, inputs=2048, outputs=5120, x8=False,
             bias=False, dtype="bf16"),
        # the output product of a small batch, with a bias, a ragged last block of outputs
        dict(name="linear-37", kind="linear", tokens=37, inputs=4096, outputs=2880, x8=True,
             bias=True, dtype="bf16"),
        # a prompt's chunk
        dict(name="linear-4096", kind="linear", tokens=4096, inputs=2048, outputs=5120, x8=True,
             bias=False, dtype="bf16"),
        # 61 decoding sequences, one token each, far into their contexts, with the heads' norm
        dict(name="rope-61", kind="rope", seqs=61, new=1, ctx=40000, ragged=True, heads=32,
             kv_heads=4, dim=128, rot=128, page=64, norm=True, interleaved=False, dtype="bf16"),
        # a prompt's chunk, interleaved pairs
        dict(name="rope-4096", kind="rope", seqs=2, new=2048, ctx=2048, ragged=False, heads=64,
             kv_heads=8, dim=64, rot=64, page=16, norm=False, interleaved=True, dtype="fp16"),
        # one sequence far into its context: the cache's bytes, split along their length
        dict(name="attn-decode-1", kind="attn", seqs=1, new=1, ctx=40001, ragged=False, heads=32,
             kv_heads=4, dim=128, page=64, window=0, sinks=False, dtype="bf16"),
        # a serving batch of unequal lengths, one token each
        dict(name="attn-decode-48", kind="attn", seqs=48, new=1, ctx=9000, ragged=True, heads=64,
             kv_heads=8, dim=64, page=16, window=0, sinks=True, dtype="bf16"),
        # drafts of a few tokens verified, a layer with a window
        dict(name="attn-verify-7", kind="attn", seqs=7, new=5, ctx=3000, ragged=True, heads=64,
             kv_heads=8, dim=64, page=32, window=128, sinks=True, dtype="fp16"),
        # prompts' ragged chunks beside each other, a few tokens to hundreds
        dict(name="attn-chunk-9", kind="attn", seqs=9, new=700, ctx=2500, ragged=True, heads=64,
             kv_heads=8, dim=64, page=16, window=0, sinks=True, dtype="bf16"),
        # a chunk of a long prompt
        dict(name="attn-chunk-4096", kind="attn", seqs=1, new=4096, ctx=8192, ragged=False,
             heads=32, kv_heads=4, dim=128, page=64, window=0, sinks=False, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "rope", "attn", "attn"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "norm":
        width = _log_int(rng, 64, 8192)
        return dict(kind=kind, tokens=_log_int(rng, 1, min(16384, 23_000_000 // width)),
                    width=width, fp8=rng.random() < 0.5, dtype=dtype)
    if kind == "linear":
        inputs, outputs = 16 * _log_int(rng, 8, 256), _log_int(rng, 64, 5120)
        return dict(kind=kind, tokens=_log_int(rng, 1, min(8192, 42_000_000_000 // (inputs * outputs))),
                    inputs=inputs, outputs=outputs, x8=rng.random() < 0.5,
                    bias=rng.random() < 0.5, dtype=dtype)
    heads, kv_heads, dim = rng.choice([(32, 4, 128), (64, 8, 64), (16, 16, 64), (12, 2, 128),
                                       (7, 1, 64), (40, 8, 128)])
    page = rng.choice([16, 32, 64, 128])
    ragged = rng.random() < 0.75
    if kind == "rope":
        new = _log_int(rng, 1, 2048)
        return dict(kind=kind, seqs=_log_int(rng, 1, max(1, min(128, 4096 // new))), new=new,
                    ctx=_log_int(rng, 1, 2000 if new > 64 else 8000), ragged=ragged, heads=heads, kv_heads=kv_heads,
                    dim=dim, rot=rng.choice([dim, dim, dim // 2, 20]), page=page,
                    norm=rng.random() < 0.5, interleaved=rng.random() < 0.5, dtype=dtype)
    new = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 4096)])
    seqs = _log_int(rng, 1, 48 if new == 1 else max(1, min(32, 4096 // new)))
    # no more pairs than the longest chunk, no more cached tokens than the largest batch
    most = min(40000, 400_000 // seqs, 48_000_000 * 32 // (seqs * new * heads))
    return dict(kind=kind, seqs=seqs, new=new, ctx=_log_int(rng, 1, max(1, most - new)),
                ragged=ragged, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                window=rng.choice([0, 0, 128, 1000]), sinks=rng.random() < 0.5, dtype=dtype)


# -- inputs -------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _lengths(c):
    """New tokens and whole length of every sequence: part of the case."""
    rng = random.Random(c["seqs"] * 1000003 + c["new"] * 1009 + c["ctx"])
    if not c["ragged"]:
        return [c["new"]] * c["seqs"], [c["new"] + c["ctx"]] * c["seqs"]
    new = [rng.randint(1, c["new"]) for _ in range(c["seqs"])]
    ctx = [rng.randint(0, c["ctx"]) for _ in range(c["seqs"])]
    new[0], ctx[-1] = c["new"], c["ctx"]
    return new, [a + b for a, b in zip(new, ctx)]


def _batch(c, g):
    """A paged cache with the batch's sequences at random pages, and the query rows."""
    dt = DTYPES[c["dtype"]]
    new, lens = _lengths(c)
    width = -(-max(lens) // c["page"]) + 1
    used = [-(-n // c["page"]) for n in lens]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
    table = [[0] * width for _ in lens]
    for row, n in zip(table, used):
        for i in range(n):
            row[i] = order.pop()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    i32 = dict(dtype=torch.int32, device="cuda")
    shape = (n_pages, c["kv_heads"], c["page"], c["dim"])
    return dict(k_pages=_randn(g, *shape, dtype=dt), v_pages=_randn(g, *shape, dtype=dt),
                table=torch.tensor(table, **i32), starts=torch.tensor(starts, **i32),
                lens=torch.tensor(lens, **i32), most_new=max(new), tokens=starts[-1])


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "norm":
        T, D = c["tokens"], c["width"]
        return dict(case=c, x=_randn(g, T, D, scale=0.7, dtype=dt), r=_randn(g, T, D, scale=3.0, dtype=dt),
                    w=(1 + _randn(g, D, scale=0.2)).to(dt))
    if c["kind"] == "linear":
        T, K, N = c["tokens"], c["inputs"], c["outputs"]
        blocks = -(-K // 128)
        s = dict(case=c, w=_randn(g, N, K, scale=100.0).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn),
                 ws=(torch.rand((-(-N // 128), blocks), generator=g, device="cuda") + 0.5) * 3e-4)
        s["bias"] = _randn(g, N, dtype=dt) if c["bias"] else None
        s["x"], s["xs"] = _randn(g, T, K, dtype=dt), None
        if c["x8"]:
            s["x"], s["xs"] = _to_fp8(s["x"].float())
        return s
    s = dict(case=c, **_batch(c, g))
    T, H, HK, D = s["tokens"], c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "attn":
        s["q"] = _randn(g, T, H, D, scale=1.5, dtype=dt)
        s["sinks"] = _randn(g, H) if c["sinks"] else None
        s["scale"] = D ** -0.5
        return s
    # the query, key and value columns of one product's output
    qkv = _randn(g, T, H + 2 * HK, D, dtype=dt)
    s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:]
    s["qw"] = (1 + _randn(g, D, scale=0.2)).to(dt) if c["norm"] else None
    s["kw"] = (1 + _randn(g, D, scale=0.2)).to(dt) if c["norm"] else None
    i = torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda")
    s["freqs"] = 150000.0 ** (-i / c["rot"])
    s["mscale"] = 1.25
    return s


# -- plain forms --------------------------------------------------------------
def _to_fp8(y):
    """y in 32 bits -> e4m3 values and a scale per 128 columns."""
    T, D = y.shape
    blocks = -(-D // 128)
    p = torch.nn.functional.pad(y, (0, blocks * 128 - D)).view(T, blocks, 128)
    most = p.abs().amax(-1).clamp_min(1e-30)
    # values halfway between two codes stay there: 448 times a value of 16 bits is exact
    q = (p * FP8_MAX / most[..., None]).view(T, blocks * 128)[:, :D].to(torch.float8_e4m3fn)
    return q.contiguous(), most / FP8_MAX


def _plain_norm(s):
    c = s["case"]
    h = (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    if c["fp8"]:
        q, scales = _to_fp8(y)
        return q, scales, h
    return y.to(h.dtype), h


def _plain_linear(s):
    x, xs, w, ws = s["x"], s["xs"], s["w"], s["ws"]
    if xs is None:
        x, xs = _to_fp8(x.float())
    N, K = w.shape
    a = x.float() * xs.repeat_interleave(128, 1)[:, :K]
    b = w.float() * ws.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = a @ b.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _places(s):
    """Sequence, index among its new tokens and position of every query row."""
    t = torch.arange(s["tokens"], device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, t, right=True) - 1
    i = t - starts[seq]
    return seq, i, s["lens"].long()[seq] - (starts[seq + 1] - starts[seq]) + i


def _plain_rope(s):
    c = s["case"]
    seq, _, pos = _places(s)
    angle = pos.double()[:, None] * s["freqs"]
    cos, sin = (angle.cos() * s["mscale"]).float()[:, None], (angle.sin() * s["mscale"]).float()[:, None]
    half = c["rot"] // 2

    def turn(x, w):
        f = x.float()
        if w is not None:
            f = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * w.float()
        if c["interleaved"]:
            a, b = f[..., 0:c["rot"]:2], f[..., 1:c["rot"]:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = f[..., :half], f[..., half:c["rot"]]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, f[..., c["rot"]:]], -1).to(x.dtype)

    page = s["table"][seq, pos // c["page"]].long()
    s["k_pages"][page, :, pos % c["page"]] = turn(s["k"], s["kw"])
    s["v_pages"][page, :, pos % c["page"]] = s["v"]
    return turn(s["q"], s["qw"]), s["k_pages"], s["v_pages"]


def _plain_attn(s):
    c = s["case"]
    H, HK, D = c["heads"], c["kv_heads"], c["dim"]
    S, Q, G = c["seqs"], s["most_new"], H // HK
    seq, i, _ = _places(s)
    table, starts, lens = s["table"].long(), s["starts"].long(), s["lens"].long()
    k = s["k_pages"][table].transpose(1, 2).reshape(S, HK, -1, D).float()
    v = s["v_pages"][table].transpose(1, 2).reshape(S, HK, -1, D).float()
    at = (starts[:-1, None] + torch.arange(Q, device="cuda")).clamp_max(s["tokens"] - 1)
    q = s["q"][at].float().view(S, Q, HK, G, D).permute(0, 2, 3, 1, 4).reshape(S, HK, G * Q, D)
    z = torch.matmul(q, k.transpose(2, 3).contiguous()).view(S, HK, G, Q, -1) * s["scale"]
    pos = ((lens - starts[1:] + starts[:-1])[:, None] + torch.arange(Q, device="cuda"))[..., None]
    j = torch.arange(k.shape[2], device="cuda")
    seen = (j <= pos) & (j < lens[:, None, None])
    if c["window"]:
        seen = seen & (j > pos - c["window"])
    z = z.masked_fill_(~seen[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True).clamp_min(-1e30)
    sink = None if s["sinks"] is None else s["sinks"].view(1, HK, G, 1, 1)
    if sink is not None:
        m = torch.maximum(m, sink)
    e = z.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    if sink is not None:
        total = total + (sink - m).exp()
    o = torch.matmul(e.view(S, HK, G * Q, -1), v).view(S, HK, G, Q, D) / total.clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(S, Q, H, D)[seq, i].to(s["q"].dtype)


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "rope": _plain_rope,
                "attn": _plain_attn}[kind](s)
    from moe_stream_amd import ops
    if kind == "norm":
        if s["case"]["fp8"]:
            return ops.add_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS, fp8=True)
        return ops.add_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
    if kind == "linear":
        return ops.linear_fp8(s["x"], s["w"], s["ws"], x_scales=s["xs"], bias=s["bias"],
                              dtype=DTYPES[s["case"]["dtype"]])
    if kind == "rope":
        q = ops.rope_cache(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"],
                           s["starts"], s["lens"], s["freqs"],
                           interleaved=s["case"]["interleaved"], mscale=s["mscale"],
                           q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
        return q, s["k_pages"], s["v_pages"]
    return ops.attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["lens"],
                          scale=s["scale"], window=s["case"]["window"], sinks=s["sinks"])


def work(case):
    c = case
    if c["kind"] == "norm":
        T, D = c["tokens"], c["width"]
        out = T * D + 4 * T * -(-D // 128) if c["fp8"] else 2 * T * D
        return {"bytes": 6 * T * D + 2 * D + out, "flops": 8 * T * D}
    if c["kind"] == "linear":
        T, K, N = c["tokens"], c["inputs"], c["outputs"]
        blocks = -(-K // 128)
        x = T * K + 4 * T * blocks if c["x8"] else 2 * T * K
        return {"bytes": x + N * K + 4 * blocks * -(-N // 128) + 2 * T * N + (2 * N if c["bias"] else 0),
                "flops": 2 * T * N * K}
    new, lens = _lengths(c)
    H, HK, D, T = c["heads"], c["kv_heads"], c["dim"], sum(new)
    if c["kind"] == "rope":
        return {"bytes": 4 * T * (H + 2 * HK) * D, "flops": 12 * T * (H + HK) * D}
    pairs = keys = 0
    for n, L in zip(new, lens):
        w = c["window"] or L
        first = L - n
        # position p sees min(p + 1, w) keys
        short = max(0, min(L, w) - first)
        pairs += short * (2 * first + short + 1) // 2 + (n - short) * w
        keys += L - max(0, first - w + 1)
    return {"bytes": 4 * T * H * D + 4 * keys * HK * D, "flops": 4 * D * H * pairs}


# -- the definitions in 64 bits -------------------------------------------------
def _quant64(y):
    n = y.shape[1]
    scales = []
    vals = []
    for a in range(0, n, 128):
        b = y[:, a:a + 128]
        top = torch.clamp(b.abs().max(dim=1).values, min=1e-30)
        scales.append(top / FP8_MAX)
        # e4m3: 3 fraction bits down to 2^-6, steps of 2^-9 below it
        r = b * FP8_MAX / top[:, None]
        e = torch.floor(torch.log2(r.abs().clamp_min(2.0 ** -6))).clamp_max(8.0)
        step = torch.exp2(e - 3)
        vals.append(torch.round(r / step) * step)
    return torch.cat(vals, 1), torch.stack(scales, 1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "norm":
        h = (s["x"].double() + s["r"].double()).to(s["x"].dtype)
        d = h.double()
        y = d / torch.sqrt((d * d).sum(1, keepdim=True) / c["width"] + EPS) * s["w"].double()
        return (*_quant64(y), h.double()) if c["fp8"] else (y, h.double())
    if c["kind"] == "linear":
        q, xs = (s["x"].double(), s["xs"].double()) if c["x8"] else _quant64(s["x"].double())
        y = torch.zeros((c["tokens"], c["outputs"]), dtype=torch.float64, device="cuda")
        col = s["ws"].double()[torch.arange(c["outputs"], device="cuda") // 128]
        for b in range(xs.shape[1]):
            part = q[:, 128 * b:128 * b + 128] @ s["w"][:, 128 * b:128 * b + 128].double().t().contiguous()
            y += part * xs[:, b:b + 1] * col[:, b]
        return y + s["bias"].double() if c["bias"] else y
    new, lens = _lengths(c)
    H, HK, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    table = s["table"].tolist()
    rows, at = [], 0
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    for n, L, pages in zip(new, lens, table):
        pos = torch.arange(L - n, L, device="cuda")
        if c["kind"] == "rope":
            turned = []
            for x, w in ((s["q"][at:at + n].double(), s["qw"]), (s["k"][at:at + n].double(), s["kw"])):
                if w is not None:
                    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
                y = x.clone()
                for f in range(c["rot"] // 2):
                    i0, i1 = (2 * f, 2 * f + 1) if c["interleaved"] else (f, f + c["rot"] // 2)
                    z = torch.polar(torch.full((n,), s["mscale"], dtype=torch.float64, device="cuda"),
                                    pos.double() * s["freqs"][f])
                    z = torch.complex(x[..., i0], x[..., i1]) * z[:, None]
                    y[..., i0], y[..., i1] = z.real, z.imag
                turned.append(y)
            rows.append(turned[0])
            where = torch.tensor(pages, device="cuda")[pos // page]
            for h in range(HK):
                kp[where, h, pos % page] = turned[1][:, h]
                vp[where, h, pos % page] = s["v"][at:at + n, h].double()
        else:
            own_pages = torch.tensor(pages[:-(-L // page)], device="cuda")
            out = torch.empty((n, H, D), dtype=torch.float64, device="cuda")
            keys = torch.arange(L, device="cuda")[None]
            hidden = keys > pos[:, None]
            if c["window"]:
                hidden |= keys <= pos[:, None] - c["window"]
            for h in range(H):
                g = h // (H // HK)
                k = kp[own_pages, g].reshape(-1, D)[:L]
                v = vp[own_pages, g].reshape(-1, D)[:L]
                z = s["q"][at:at + n, h].double() @ k.t().contiguous() * s["scale"]
                z[hidden] = -math.inf
                if s["sinks"] is not None:
                    z = torch.cat([z, s["sinks"][h].double().expand(n, 1)], 1)
                p = torch.softmax(z, 1)[:, :L]
                out[:, h] = p @ v
            rows.append(out)
        at += n
    y = torch.cat(rows)
    return (y, kp, vp) if c["kind"] == "rope" else y
