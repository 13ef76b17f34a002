"""The operators of a layer's prompt path, as cases to time and to check.

Three operators that a serving program calls next to paged attention:

* "rotate": per-head RMS norm of the projected queries and keys, rotation by position
  (half or interleaved pairs, part of the head, scaled frequencies) and the write of keys
  and values into the paged cache, quantised when the cache is FP8.
* "attend": causal attention of packed prompts straight from contiguous keys and values,
  with grouped heads, a cached prefix per sequence and any number of new tokens from one on.
* "readback": the keys and values of cached sequences, gathered through their block tables
  and dequantised into packed rows.

`own` false computes the plain form with elementary torch operations; `own` true makes the
calls of the paged_attn_b200 package.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
HEADS = (32, 64, 80, 96, 112, 120, 128, 192, 256)


def listed():
    return [
        # one sequence generating: a single token between two projections
        dict(name="rotate-step-1", op="rotate", tokens=1, hq=16, hkv=8, head=128, dims=128, inter=False,
             scaling="none", factor=1.0, norm=True, fp8=False, block=16, f16=False, far=1777, keep_k=False),
        # one decode step of a batch of 64 sequences
        dict(name="rotate-decode-64", op="rotate", tokens=64, hq=32, hkv=8, head=128, dims=128, inter=False,
             scaling="none", factor=1.0, norm=True, fp8=False, block=16, f16=False, far=8000, keep_k=False),
        # a prompt of 8192 tokens at positions beyond the trained length, keys kept for the attention
        dict(name="rotate-prompt-8192", op="rotate", tokens=8192, hq=32, hkv=8, head=128, dims=128, inter=False,
             scaling="yarn", factor=4.0, norm=True, fp8=False, block=16, f16=False, far=120000, keep_k=True),
        # an odd chunk into an FP8 cache of 32-token blocks, half the head rotated in interleaved pairs
        dict(name="rotate-chunk-fp8", op="rotate", tokens=2049, hq=64, hkv=8, head=128, dims=64, inter=True,
             scaling="linear", factor=8.0, norm=False, fp8=True, block=32, f16=True, far=30000, keep_k=True),
        # a batch of short requests, seven query heads to a key head, small heads
        dict(name="attend-short", op="attend", seqs=12, lo=1, hi=200, prefix_lo=0, prefix_hi=0, lens=3,
             hq=14, hkv=2, head=64, f16=False, softcap=1.0),
        # one long prompt
        dict(name="attend-prompt-8192", op="attend", seqs=1, lo=8192, hi=8192, prefix_lo=0, prefix_hi=0, lens=0,
             hq=32, hkv=8, head=128, f16=False, softcap=1.0),
        # prompts of ragged lengths admitted together
        dict(name="attend-packed", op="attend", seqs=7, lo=700, hi=2500, prefix_lo=0, prefix_hi=0, lens=5,
             hq=32, hkv=8, head=128, f16=True, softcap=1.0),
        # two prefill chunks of 1024 tokens, each over a prefix of 4096 read back from the cache
        dict(name="attend-chunks", op="attend", seqs=2, lo=1024, hi=1024, prefix_lo=4096, prefix_hi=4096, lens=1,
             hq=32, hkv=8, head=128, f16=False, softcap=1.0),
        # single tokens and short drafts over long contiguous contexts
        dict(name="attend-tokens", op="attend", seqs=8, lo=1, hi=5, prefix_lo=4000, prefix_hi=16000, lens=2,
             hq=64, hkv=8, head=128, f16=False, softcap=1.0),
        # the prefix of one sequence
        dict(name="readback-one", op="readback", seqs=1, lo=700, hi=700, skip=0, lens=1, hkv=8, head=128,
             fp8=False, block=16, f16=False),
        # the prefixes of a batch, 16-bit
        dict(name="readback-batch", op="readback", seqs=8, lo=2000, hi=8192, skip=0, lens=4, hkv=8, head=128,
             fp8=False, block=16, f16=False),
        # a range of tokens out of an FP8 cache of 32-token blocks
        dict(name="readback-fp8", op="readback", seqs=9, lo=1000, hi=8192, skip=333, lens=6, hkv=8, head=128,
             fp8=True, block=32, f16=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _geometry(rng, fp8):
    """Head size, block size: what a cache of that kind can be built with."""
    if fp8:
        return 128, rng.choice((16, 32))
    head = rng.choice(HEADS + (64, 128, 128, 128))
    return head, rng.choice((8, 16, 32)) if head == 128 else rng.choice((16, 32)) if head < 128 else 16


def draw(rng):
    op = rng.choice(("rotate", "attend", "attend", "readback"))
    if op == "rotate":
        fp8 = rng.random() < 0.3
        head, block = _geometry(rng, fp8)
        hkv = rng.choice((1, 2, 3, 4, 8))
        dims = head if rng.random() < 0.6 else 2 * rng.randint(1, head // 2)
        scaling = rng.choice(("none", "none", "linear", "bands", "yarn"))
        return dict(op=op, tokens=_log(rng, 1, 6000), hq=hkv * rng.choice((1, 2, 3, 4, 5, 7, 8)), hkv=hkv, head=head,
                    dims=dims, inter=rng.random() < 0.4, scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0, 32.0)),
                    norm=rng.random() < 0.6, fp8=fp8, block=block, f16=rng.random() < 0.4,
                    far=_log(rng, 1, 1000000), keep_k=rng.random() < 0.5)
    if op == "attend":
        head = rng.choice(HEADS + (64, 128, 128, 128, 128))
        hkv = rng.choice((1, 2, 4, 8))
        group = rng.choice((1, 2, 3, 4, 5, 7, 8, 12))
        group = max(1, min(group, 64 * 128 // (head * hkv)))
        form = rng.choice(("prompts", "chunks", "tokens"))
        seqs = rng.randint(1, 10)
        if form == "prompts":
            hi = _log(rng, 2, 5000)
            lo, p_lo, p_hi = rng.randint(max(1, hi // 4), hi), 0, 0
        elif form == "chunks":
            hi, p_hi = _log(rng, 16, 1500), _log(rng, 100, 6000)
            lo, p_lo = rng.randint(max(1, hi // 3), hi), rng.randint(0, p_hi)
        else:
            hi, p_hi = rng.randint(1, 6), _log(rng, 100, 30000)
            lo, p_lo = 1, rng.randint(p_hi // 4, p_hi)
        # no more score entries than the long prompt has
        while seqs > 1 and seqs * hkv * group * hi * (hi + p_hi) > 32 * 8192 * 8192 * 0.6:
            seqs -= 1
        if hkv * group * hi * (hi + p_hi) * head > 32 * 8192 * 8192 * 64:
            hkv, group = 2, 2
        return dict(op=op, seqs=seqs, lo=lo, hi=hi, prefix_lo=p_lo, prefix_hi=p_hi, lens=rng.randint(0, 1 << 20),
                    hq=hkv * group, hkv=hkv, head=head, f16=rng.random() < 0.4,
                    softcap=rng.choice((1.0, 1.0, 1.0, 30.0)))
    fp8 = rng.random() < 0.4
    head, block = _geometry(rng, fp8)
    hi = _log(rng, 1, 8000)
    return dict(op=op, seqs=rng.randint(1, 8), lo=rng.randint(max(1, hi // 4), hi), hi=hi, skip=rng.choice((0, 0, 16, 5, 1001)),
                lens=rng.randint(0, 1 << 20), hkv=rng.choice((1, 2, 4, 8)), head=head, fp8=fp8, block=block,
                f16=rng.random() < 0.4)


# ---- what a case says about its lengths -------------------------------------------------
def _lens(case):
    """(new tokens, all tokens) of each sequence."""
    r = random.Random(case["lens"])
    q = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    if case["op"] == "readback":
        return q, q
    return q, [n + r.randint(case["prefix_lo"], case["prefix_hi"]) for n in q]


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def work(case):
    d, hkv = case["head"], case["hkv"]
    if case["op"] == "rotate":
        t, hq = case["tokens"], case["hq"]
        read = t * (hq + 2 * hkv) * d * 2 + t * 12 + (4 * d if case["norm"] else 0)
        written = t * hq * d * 2 + t * 2 * hkv * d * (1 if case["fp8"] else 2)
        written += t * hkv * d * 2 if case["keep_k"] else 0
        return {"bytes": read + written, "flops": t * (hq + hkv) * (3 * case["dims"] + (4 * d if case["norm"] else 0))}
    q, kv = _lens(case)
    if case["op"] == "attend":
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, kv))
        return {"bytes": 2 * d * (2 * sum(q) * case["hq"] + 2 * sum(kv) * hkv), "flops": 4 * d * case["hq"] * pairs}
    t = sum(q)
    return {"bytes": t * hkv * d * 2 * (3 if case["fp8"] else 4) + 4 * t // case["block"], "flops": 0}


# ---- inputs -----------------------------------------------------------------------------
def _normal(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _frequencies(case):
    """Radians per position of each pair, and what cosine and sine are multiplied by (64 bits)."""
    half = case["dims"] // 2
    base, factor, trained = 1e6, case["factor"], 4096.0
    f = base ** (-torch.arange(half, dtype=torch.float64) / half)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "bands":  # long waves are slowed down, short ones kept, in between a blend
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    if case["scaling"] == "yarn":  # a ramp over the pair's index between 32 turns and one turn
        where = lambda turns: half * math.log(trained / (turns * 2 * math.pi)) / math.log(base)  # noqa: E731
        lo, hi = max(math.floor(where(32.0)), 0), min(math.ceil(where(1.0)), case["dims"] - 1)
        slow = ((torch.arange(half, dtype=torch.float64) - lo) / (max(hi - lo, 0.001))).clamp(0, 1)
        return f / factor * slow + f * (1 - slow), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _pools(case, blocks, g=None):
    """Key and value pool of one layer; with a generator, as a cache that holds tokens."""
    d, bs, hkv = case["head"], case["block"], case["hkv"]
    x = 16 if case["fp8"] else 8
    shapes = (blocks, hkv, d // x, bs, x), (blocks, hkv, d, bs)
    if case["fp8"]:
        if g is None:
            return [torch.zeros(s, dtype=torch.uint8, device="cuda") for s in shapes]
        return [(torch.randn(s, generator=g, device="cuda") * 30).clamp(-240, 240).to(F8).view(torch.uint8) for s in shapes]
    t = torch.float16 if case["f16"] else torch.bfloat16
    if g is None:
        return [torch.zeros(s, dtype=t, device="cuda") for s in shapes]
    return [_normal(g, *s, dtype=t) for s in shapes]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t16 = torch.float16 if case["f16"] else torch.bfloat16
    d, hkv = case["head"], case["hkv"]
    s = dict(case=dict(case), op=case["op"], dtype=t16)
    if case["op"] == "rotate":
        t, hq = case["tokens"], case["hq"]
        bs = case["block"]
        # the three projections' outputs, as one matrix product leaves them
        qkv = _normal(g, t, hq + 2 * hkv, d, dtype=t16, scale=1.5)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["qw"] = s["kw"] = None
        if case["norm"]:
            s["qw"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(t16)
            s["kw"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(t16)
        blocks = -(-t // bs) + 3
        order = torch.randperm(blocks, generator=g, device="cuda")
        at = torch.arange(t, device="cuda")
        s["slots"] = order[at // bs] * bs + at % bs
        s["positions"] = (case["far"] + at).to(torch.int32)
        s["q_out"] = torch.empty(t, hq, d, dtype=t16, device="cuda")
        s["k_out"] = torch.empty(t, hkv, d, dtype=t16, device="cuda") if case["keep_k"] else None
        s["pools"] = _pools(case, blocks)
        s["scales"] = (1 / 16, 1 / 8)
        f, s["gain"] = _frequencies(case)
        s["freq"] = f.cuda()
    elif case["op"] == "attend":
        q, kv = _lens(case)
        hq = case["hq"]
        # queries and keys as they leave their norms: logits of a few units
        s["q"] = _normal(g, sum(q), hq, d, dtype=t16, scale=1.4)
        s["k"] = _normal(g, sum(kv), hkv, d, dtype=t16, scale=1.4)
        s["v"] = _normal(g, sum(kv), hkv, d, dtype=t16)
        s["cu_q"], s["cu_kv"] = _cu(q), _cu(kv)
        s["out"] = torch.empty(sum(q), hq, d, dtype=t16, device="cuda")
        s["scale"] = d ** -0.5
        s["lens_q"], s["lens_kv"] = torch.tensor(q, device="cuda"), torch.tensor(kv, device="cuda")
        s["max_q"], s["max_kv"] = max(q), max(kv)
        s["pools"] = None
    else:
        lens, _ = _lens(case)
        bs, skip = case["block"], case["skip"]
        per = [-(-(n + skip) // bs) for n in lens]
        order = torch.randperm(sum(per) + 5, generator=g, device="cuda").to(torch.int32)
        s["tables"] = torch.zeros(len(lens), max(per), dtype=torch.int32, device="cuda")
        for i, n in enumerate(per):
            s["tables"][i, :n] = order[sum(per[:i]):sum(per[:i]) + n]
        s["cu"] = _cu(lens)
        s["starts"] = np.full(len(lens), skip, dtype=np.int32)
        s["lens"] = torch.tensor(lens, device="cuda")
        s["pools"] = _pools(case, sum(per) + 5, g)
        s["scales"] = (1 / 16, 1 / 8)
        s["key"] = torch.empty(sum(lens), hkv, d, dtype=t16, device="cuda")
        s["value"] = torch.empty(sum(lens), hkv, d, dtype=t16, device="cuda")
    if own:
        _handles(s)
    return s


def _handles(s):
    """The cache handle, plan and workspace that a serving program keeps."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if os.path.join(root, "mlx-node_b200") not in sys.path:
        sys.path.insert(0, os.path.join(root, "mlx-node_b200"))
    import paged_attn_b200 as pa
    c = s["case"]
    fp8 = c.get("fp8", False)
    if s["pools"] is not None:
        s["cache"] = pa.PagedCache(c["block"], s["pools"][0].shape[0], c["head"], c["hkv"], dtype=0 if c["f16"] else 1,
                                   key_pools=s["pools"][:1], value_pools=s["pools"][1:], fp8=fp8)
        if fp8:
            s["cache"].set_kv_scales(*s["scales"])
    else:
        s["cache"] = pa.PagedCache(16, 4, c["head"], c["hkv"], dtype=0 if c["f16"] else 1)
    if s["op"] == "rotate":
        s["plan"] = pa.RopePlan(c["dims"], 1e6, interleaved=c["inter"], scaling=c["scaling"], factor=c["factor"],
                                original_max_position=4096)
    if s["op"] == "attend":
        s["ws_bytes"] = s["cache"].prompt_workspace_bytes()
        s["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device="cuda")


# ---- one pass ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        cache, d = s["cache"], c["head"]
        if s["op"] == "rotate":
            row = (c["hq"] + 2 * c["hkv"]) * d
            cache.rope_norm_and_cache(s["plan"], s["q_out"], s["k_out"], s["q"], s["k"], s["v"], s["qw"], s["kw"], 1e-6,
                                      s["positions"], s["slots"], c["tokens"], c["hq"], q_stride=row, k_stride=row,
                                      v_stride=row)
        elif s["op"] == "attend":
            cache.prompt_attention(s["out"], s["q"], s["k"], s["v"], s["cu_q"], s["cu_kv"], c["seqs"], c["hq"],
                                   s["scale"], s["ws"], s["ws_bytes"], softcap=c["softcap"])
        else:
            cache.gather(s["key"], s["value"], s["tables"], s["starts"], s["cu"], c["seqs"], s["tables"].shape[1])
    elif s["op"] == "rotate":
        _plain_rotate(s)
    elif s["op"] == "attend":
        s["out"] = _plain_attend(s)
    else:
        s["key"], s["value"] = _plain_readback(s)
    if s["op"] == "attend":
        return {"out": s["out"]}
    if s["op"] == "readback":
        return {"key": s["key"], "value": s["value"]}
    # an FP8 cache's bytes are E4M3 numbers: the values they stand for, before the scale
    pools = [p.view(F8) if c["fp8"] else p for p in s["pools"]]
    return {"q": s["q_out"], "k": s["k_out"], "key_pool": pools[0], "value_pool": pools[1]}


def _plain_rotate(s):
    c, t16 = s["case"], s["dtype"]
    dims, half = c["dims"], c["dims"] // 2
    angle = s["positions"].double()[:, None] * s["freq"]  # 64 bits: far positions
    cos = (angle.cos() * s["gain"]).float()[:, None]
    sin = (angle.sin() * s["gain"]).float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        r, rest = x[..., :dims], x[..., dims:]
        a, b = (r[..., 0::2], r[..., 1::2]) if c["inter"] else (r[..., :half], r[..., half:])
        a, b = a * cos - b * sin, b * cos + a * sin
        r = torch.stack((a, b), -1).flatten(-2) if c["inter"] else torch.cat((a, b), -1)
        return torch.cat((r, rest), -1).to(t16)

    s["q_out"] = turned(s["q"], s["qw"])
    k = turned(s["k"], s["kw"])
    if c["keep_k"]:
        s["k_out"] = k
    v = s["v"]
    if c["fp8"]:
        k = (k.float() / s["scales"][0]).to(F8).view(torch.uint8)
        v = (v.float() / s["scales"][1]).to(F8).view(torch.uint8)
    kp, vp = s["pools"]
    block, off = s["slots"] // c["block"], s["slots"] % c["block"]
    kp[block, :, :, off] = k.unflatten(-1, (-1, kp.shape[-1]))
    vp[block, :, :, off] = v


def _plain_attend(s):
    """Every sequence padded to the longest: scores, mask, softmax and the weighted sum."""
    c = s["case"]
    hkv, d = c["hkv"], c["head"]
    at_q = torch.arange(s["max_q"], device="cuda")
    at_kv = torch.arange(s["max_kv"], device="cuda")
    lq, lkv = s["lens_q"], s["lens_kv"]
    row_q = (lq.cumsum(0) - lq)[:, None] + torch.minimum(at_q, lq[:, None] - 1)
    row_kv = (lkv.cumsum(0) - lkv)[:, None] + torch.minimum(at_kv, lkv[:, None] - 1)
    q = s["q"].float()[row_q].unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4)  # [S, Hkv, G, Lq, D]
    k = s["k"].float()[row_kv].permute(0, 2, 3, 1)[:, :, None]  # [S, Hkv, 1, D, Lkv]
    v = s["v"].float()[row_kv].permute(0, 2, 1, 3)[:, :, None]
    seqs, lq_max = q.shape[0], q.shape[3]
    x = (q.flatten(2, 3) @ k[:, :, 0]).unflatten(2, (-1, lq_max))
    x *= s["scale"]
    if c["softcap"] != 1.0:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    limit = (lkv - lq)[:, None] + at_q  # the last key a query sees
    x.masked_fill_((at_kv > limit[:, :, None])[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.flatten(2, 3) @ v[:, :, 0]).unflatten(2, (-1, lq_max)) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, lq_max, -1, d)
    return o[at_q < lq[:, None]].to(s["dtype"])


def _plain_readback(s):
    c = s["case"]
    lens = s["lens"]
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), lens, output_size=int(s["cu"][-1]))
    at = torch.arange(int(s["cu"][-1]), device="cuda") - (lens.cumsum(0) - lens)[seq] + c["skip"]
    block, off = s["tables"][seq, at // c["block"]].long(), at % c["block"]
    k = s["pools"][0][block, :, :, off]  # [T, Hkv, D/x, x]
    v = s["pools"][1][block, :, :, off]
    if c["fp8"]:
        k, v = (p.view(F8).float() * w for p, w in zip((k, v), s["scales"]))
    return k.flatten(2).to(s["dtype"]), v.to(s["dtype"])


# ---- the definitions in 64 bits ------------------------------------------------------------
def exact(case, seed):
    s = prepare_inputs(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(case, s)
    if case["op"] == "attend":
        return {"out": _exact_attend(case, s)}
    return _exact_readback(case, s)


def prepare_inputs(case, seed):
    """The inputs alone, whatever `own` says."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _exact_rotate(case, s):
    """Each pair as a complex number times exp(i * position * frequency)."""
    d, dims = case["head"], case["dims"]
    j = torch.arange(dims // 2, device="cuda")
    first, second = (2 * j, 2 * j + 1) if case["inter"] else (j, j + dims // 2)
    turn = torch.polar(torch.full((), s["gain"], dtype=torch.float64, device="cuda").expand(case["tokens"], dims // 2),
                       torch.outer(s["positions"].double(), s["freq"]))

    def one(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k, v = one(s["q"], s["qw"]), one(s["k"], s["kw"]), s["v"].double()
    kept = k if case["keep_k"] else None
    ks, vs = s["scales"] if case["fp8"] else (1.0, 1.0)
    kp, vp = (torch.zeros(p.shape, dtype=torch.float64, device="cuda") for p in s["pools"])
    bs, x = case["block"], kp.shape[-1]
    block, off = torch.div(s["slots"], bs, rounding_mode="floor"), torch.remainder(s["slots"], bs)
    for h in range(case["hkv"]):
        for c in range(d // x):
            kp[block, h, c, off] = k[:, h, c * x:(c + 1) * x] / ks
        vp[block, h, :, off] = v[:, h] / vs
    return {"q": q, "k": kept, "key_pool": kp, "value_pool": vp}


def _exact_attend(case, s):
    hkv, g = case["hkv"], case["hq"] // case["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["seqs"]):
        a, b, m, n = (int(v) for v in (s["cu_q"][i], s["cu_q"][i + 1], s["cu_kv"][i], s["cu_kv"][i + 1]))
        sees = torch.arange(n - m, device="cuda")[None] <= torch.arange(n - m - (b - a), n - m, device="cuda")[:, None]
        for h in range(case["hq"]):
            z = s["q"][a:b, h].double() @ s["k"][m:n, h // g].double().T * s["scale"]
            if case["softcap"] != 1.0:
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            z = torch.where(sees, z, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
            out[a:b, h] = torch.softmax(z, -1) @ s["v"][m:n, h // g].double()
    return out


def _exact_readback(case, s):
    keys, values = [], []
    ks, vs = s["scales"] if case["fp8"] else (1.0, 1.0)
    kp, vp = ((p.view(F8) if case["fp8"] else p).double() for p in s["pools"])
    for i in range(case["seqs"]):
        n, skip = int(s["cu"][i + 1] - s["cu"][i]), case["skip"]
        per = -(-(n + skip) // case["block"])
        ids = s["tables"][i, :per].long()
        k = kp[ids].permute(0, 3, 1, 2, 4).reshape(per * case["block"], case["hkv"], case["head"])
        v = vp[ids].permute(0, 3, 1, 2).reshape(per * case["block"], case["hkv"], case["head"])
        keys.append(k[skip:skip + n] * ks)
        values.append(v[skip:skip + n] * vs)
    return {"key": torch.cat(keys), "value": torch.cat(values)}
