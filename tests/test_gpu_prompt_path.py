"""GPU tests of the prompt path - rotation + cache write (pa_rope_norm_and_cache), cache read-back
(pa_gather_cache) and packed prompt attention (pa_prompt_attention) - against plain
statements in 64 bits, alone and in the run a serving program makes of them.

Tolerances.  `u` is half a step of the output type relative to a value (eps / 2).

* rotation: computed in fp32 and rounded once, so |got - exact| <= u |exact| + 2^-19 (|a| + |b|),
  (a, b) the normalised pair: the mean of squares (a sum of at most 256 products in fp32, error
  below 2^-20 of it whatever the order for the tree the kernels use), a root, a division and
  two products, sine and cosine to about 2^-22, three more products; plus half the smallest
  number of the type.
* attention: probabilities are rounded to the 16-bit type for the tensor cores (u each) and
  the output once more (u): |got - exact| <= (u + 2^-13) (sum p|v| + |exact|), where 2^-13
  covers fp32 logits of magnitude up to a few tens (a dot product's rounding, 2^-24 of
  sum |q k|, enters the probability as a relative error) and exp2; an f16 probability below
  2^-14 is off by up to 2^-25 absolute instead, relative to a sum of at least one.
* read-back: the bytes are moved, or decoded, scaled in fp32 and rounded once: exact.
"""
import math

import numpy as np
import pytest
import torch

import paged_attn_b200 as pa
from gpu_util import to_bits

pytestmark = pytest.mark.gpu

HEADS = (32, 64, 80, 96, 112, 120, 128, 192, 256)
T16 = {False: torch.bfloat16, True: torch.float16}


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, t=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)


# ---- rotation + cache write -----------------------------------------------------------------
def rotate_exact(x, w, eps, positions, freq, gain, dims, inter):
    """(exact rows in 64 bits, magnitude |a| + |b| of each element's pair)."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    half = dims // 2
    j = torch.arange(half, device=x.device)
    a, b = (2 * j, 2 * j + 1) if inter else (j, j + half)
    # 64 bits hold a position times a frequency to 2^-21 of a turn at 2^31; reduce in turns
    angle = torch.outer(positions.double(), torch.tensor(freq, dtype=torch.float64, device=x.device))
    c, s = torch.cos(angle)[:, None] * gain, torch.sin(angle)[:, None] * gain
    out, mag = y.clone(), y.abs()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    m = (y[..., a].abs() + y[..., b].abs()) * gain
    mag[..., a] = m
    mag[..., b] = m
    return out, mag


def check_rotated(got, ref, mag, what):
    t = got.dtype
    tiny = 2.0 ** -25 if t == torch.float16 else 2.0 ** -134
    bound = half_step(t) * ref.abs() + 2.0 ** -19 * mag + tiny
    bad = (got.double() - ref).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} elements beyond the bound, worst " \
                          f"{((got.double() - ref).abs() / bound).max().item():.2f} of it"


class Rotate:
    def __init__(self, tokens, hq, hkv, head, dims, inter=False, norm=True, fp8=False, block=16, f16=False, far=0,
                 keep_k=True, write=True, seed=0, pad=0, **plan):
        g = gen(seed)
        t = T16[f16]
        self.t, self.norm, self.dims, self.inter, self.keep_k, self.write = tokens, norm, dims, inter, keep_k, write
        self.hq, self.hkv, self.head, self.block, self.fp8 = hq, hkv, head, block, fp8
        self.qkv = randn(g, tokens, hq + 2 * hkv + pad, head, t=t, scale=1.5)
        self.q, self.k, self.v = self.qkv[:, :hq], self.qkv[:, hq:hq + hkv], self.qkv[:, hq + hkv:hq + 2 * hkv]
        self.row = (hq + 2 * hkv + pad) * head
        self.qw = (1 + 0.2 * torch.randn(head, generator=g, device="cuda")).to(t) if norm else None
        self.kw = (1 + 0.2 * torch.randn(head, generator=g, device="cuda")).to(t) if norm else None
        self.positions = (far + torch.arange(tokens, device="cuda")).to(torch.int32)
        blocks = -(-tokens // block) + 2
        order = torch.randperm(blocks, generator=g, device="cuda")
        at = torch.arange(tokens, device="cuda")
        self.slots = order[at // block] * block + at % block
        x = 16 if fp8 else 8
        shapes = ((blocks, hkv, head // x, block, x), (blocks, hkv, head, block))
        pool_t = torch.uint8 if fp8 else t
        self.pools = [torch.full(s, 0x7F if fp8 else float("nan"), dtype=pool_t, device="cuda") for s in shapes]
        self.cache = pa.PagedCache(block, blocks, head, hkv, dtype=0 if f16 else 1, key_pools=self.pools[:1],
                                   value_pools=self.pools[1:], fp8=fp8)
        if fp8:
            self.cache.set_kv_scales(1 / 16, 1 / 8)
        self.plan = pa.RopePlan(dims, 1e6, interleaved=inter, original_max_position=4096, **plan)
        self.q_out = torch.full((tokens + 1, hq, head), 7.0, dtype=t, device="cuda")
        self.k_out = torch.full((tokens + 1, hkv, head), 7.0, dtype=t, device="cuda") if keep_k else None

    def run(self, stream=0):
        self.cache.rope_norm_and_cache(
            self.plan, self.q_out, self.k_out, self.q, self.k, self.v if self.write else None, self.qw, self.kw, 1e-6,
            self.positions, self.slots if self.write else None, self.t, self.hq, q_stride=self.row, k_stride=self.row,
            v_stride=self.row, stream=stream)

    def check(self):
        torch.cuda.synchronize()
        self.cache.check_errors()
        f, gain = self.plan.frequencies()
        ref, mag = rotate_exact(self.q, self.qw, 1e-6, self.positions, f, gain, self.dims, self.inter)
        check_rotated(self.q_out[:-1], ref, mag, "queries")
        assert (self.q_out[-1] == 7.0).all()
        ref, mag = rotate_exact(self.k, self.kw, 1e-6, self.positions, f, gain, self.dims, self.inter)
        if self.keep_k:
            check_rotated(self.k_out[:-1], ref, mag, "keys")
            assert (self.k_out[-1] == 7.0).all()
        # the pool: what the plain cache write makes of the rotated keys and the values
        want = [torch.full_like(p, 0x7F if self.fp8 else float("nan")) for p in self.pools]
        other = pa.PagedCache(self.block, want[0].shape[0], self.head, self.hkv,
                              dtype=0 if self.q.dtype == torch.float16 else 1, key_pools=want[:1], value_pools=want[1:],
                              fp8=self.fp8)
        if self.fp8:
            other.set_kv_scales(1 / 16, 1 / 8)
        if self.write:
            if self.keep_k:
                k = self.k_out
            else:  # the same call with the keys kept
                k = torch.empty(self.t, self.hkv, self.head, dtype=self.q.dtype, device="cuda")
                q = torch.empty_like(self.q_out)
                self.cache.rope_norm_and_cache(self.plan, q, k, self.q, self.k, None, self.qw, self.kw, 1e-6, self.positions,
                                               None, self.t, self.hq, q_stride=self.row, k_stride=self.row)
                check_rotated(k, ref, mag, "keys")
            other.reshape_and_cache(k, self.v, self.slots, self.t, self.hkv * self.head, self.row)
        torch.cuda.synchronize()
        for p, w in zip(self.pools, want):
            as_int = torch.uint8 if self.fp8 else torch.int16
            assert torch.equal(p.view(as_int), w.view(as_int)), "pool differs from the plain write"


@pytest.mark.parametrize("head", HEADS)
@pytest.mark.parametrize("inter", [False, True])
def test_rotate_head_sizes(cuda_device, head, inter):
    for tokens, hq, hkv, dims, f16 in ((1, 4, 2, head, False), (37, 6, 2, head // 2 // 2 * 2, True), (130, 5, 1, 2, False),
                                       (67, 7, 1, head - 2, True)):
        r = Rotate(tokens, hq, hkv, head, dims, inter=inter, f16=f16, seed=head + tokens)
        r.run()
        r.check()


@pytest.mark.parametrize("tokens", [1, 2, 3, 15, 16, 17, 64, 255, 1000, 4099])
@pytest.mark.parametrize("block", [8, 16, 32])
def test_rotate_lengths_and_blocks(cuda_device, tokens, block):
    r = Rotate(tokens, 32, 8, 128, 128, block=block, far=5, seed=tokens, keep_k=tokens % 2 == 1, pad=tokens % 3)
    r.run()
    r.check()


@pytest.mark.parametrize("tokens", [1, 19, 513])
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("f16", [False, True])
def test_rotate_fp8(cuda_device, tokens, block, f16):
    r = Rotate(tokens, 8, 2, 128, 64, inter=True, norm=False, fp8=True, block=block, f16=f16, seed=tokens,
               scaling="linear", factor=8.0)
    r.run()
    r.check()


@pytest.mark.parametrize("plan", [dict(scaling="none"), dict(scaling="linear", factor=4.0),
                                  dict(scaling="bands", factor=8.0), dict(scaling="yarn", factor=32.0),
                                  dict(scaling="none", attention_factor=0.25)])
@pytest.mark.parametrize("far", [0, 131072, 10_000_000])
def test_rotate_scalings_and_far_positions(cuda_device, plan, far):
    r = Rotate(65, 16, 4, 128, 96, far=far, norm=far == 0, seed=3, **plan)
    r.run()
    r.check()


def test_rotate_extreme_positions(cuda_device):
    """The 64-bit reference is reduced in turns, exactly, for the positions an int32 ends at."""
    from fractions import Fraction
    r = Rotate(4, 4, 2, 64, 64, norm=False, seed=5)
    pos = [2 ** 31 - 1, -(2 ** 31), -1, 2 ** 31 - 12345]
    r.positions = torch.tensor(pos, dtype=torch.int32, device="cuda")
    r.run()
    torch.cuda.synchronize()
    f, _ = r.plan.frequencies()
    two_pi = Fraction(884279719003555, 140737488355328)  # double nearest 2 pi: 1e-16 relative, 2^-22 turns at 2^31
    angle = torch.tensor([[float((Fraction(x) * p / two_pi) % 1) * 2 * math.pi for x in f] for p in pos],
                         dtype=torch.float64, device="cuda")
    y = r.q.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    ref = torch.cat((y[..., :32] * c - y[..., 32:] * s, y[..., 32:] * c + y[..., :32] * s), -1)
    mag = (y[..., :32].abs() + y[..., 32:].abs()).repeat(1, 1, 2)
    # the double frequencies are 2^-53 off: 2^31 * 2^-53 radians, 2^-22, on top of the bound's own
    check_rotated(r.q_out[:-1], ref, mag * (1 + 2.0 ** -2), "queries")


def test_rotate_in_place_and_without_write(cuda_device):
    a = Rotate(33, 8, 2, 96, 40, seed=9, write=False)
    a.run()
    a.check()
    b = Rotate(33, 8, 2, 96, 40, seed=9, write=False)
    b.cache.rope_norm_and_cache(b.plan, b.q, b.k, b.q, b.k, None, b.qw, b.kw, 1e-6, b.positions, None, 33, 8,
                                q_stride=b.row, q_out_stride=b.row, k_stride=b.row, k_out_stride=b.row)
    torch.cuda.synchronize()
    assert torch.equal(b.q, a.q_out[:-1]) and torch.equal(b.k, a.k_out[:-1])


def test_rotate_skipped_and_bad_slots(cuda_device):
    r = Rotate(40, 4, 2, 128, 128, seed=1)
    before = [p.clone() for p in r.pools]
    good = r.slots.clone()
    r.slots[5] = -1
    r.slots[17] = r.pools[0].shape[0] * 16
    r.slots[18] = 2 ** 62
    r.run()
    torch.cuda.synchronize()
    with pytest.raises(pa.PagedAttnError) as e:
        r.cache.check_errors()
    assert e.value.status == 4
    r.cache.check_errors()
    for i in (5, 17, 18):
        blk, off = int(good[i]) // 16, int(good[i]) % 16
        assert torch.equal(r.pools[1][blk, :, :, off].view(torch.int16), before[1][blk, :, :, off].view(torch.int16))
        assert torch.equal(r.pools[0][blk, :, :, off].view(torch.int16), before[0][blk, :, :, off].view(torch.int16))
    r.slots = good
    r.run()
    r.check()


def test_rotate_fp8_overflow_switches_the_cache_to_exact(cuda_device):
    """A key that leaves E4M3's range sets the cache's flag, as the plain write does, and the
    attention then reads the byte as infinity."""
    r = Rotate(16, 2, 1, 128, 128, norm=False, fp8=True, seed=2)
    r.cache.fp8_set_exact_decode(False)
    r.v[3, 0, 7] = 1000.0
    r.run()
    r.check()
    tables = torch.tensor([[int(r.slots[0]) // 16]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([16], dtype=torch.int32, device="cuda")
    out = torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda")
    n = r.cache.workspace_bytes()
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    r.cache.decode(out, r.q_out, tables, lens, 1, 2, 1, 0.1, ws, n)
    torch.cuda.synchronize()
    byte = r.pools[1][int(r.slots[3]) // 16, 0, 7, int(r.slots[3]) % 16].item()
    if byte & 0x78 == 0x78:
        assert not torch.isfinite(out[0, :, 7]).any()


@pytest.mark.parametrize("f16", [False, True])
def test_rotate_fp8_bytes_of_every_element(cuda_device, f16):
    """Every 16-bit pattern, under scales that divide exactly and scales that do not: the bytes of
    the plain cache write, which are pinned to the oracle elsewhere."""
    t = T16[f16]
    bits = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(t)
    x = bits[torch.randperm(65536, generator=gen(1), device="cuda")].view(256, 2, 128)
    x = torch.cat((x, bits.view(256, 2, 128)))  # mixed and sorted neighbours
    n = x.shape[0]
    slots = torch.arange(n, device="cuda")
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    q = torch.zeros(n, 2, 128, dtype=t, device="cuda")
    plan = pa.RopePlan(2, 1e4)
    for ks, vs in ((1.0, 0.0371), (1 / 16, 3.0), (1e-3, 7e4), (1e-30, 1e30), (1.1, 0.9999999), (2.0 ** -61, 2.0 ** 61)):
        pools = [torch.zeros(n // 16, 2, 8, 16, 16, dtype=torch.uint8, device="cuda") for _ in range(4)]
        caches = []
        for i in (0, 2):
            caches.append(pa.PagedCache(16, n // 16, 128, 2, dtype=0 if f16 else 1, key_pools=pools[i:i + 1],
                                        value_pools=pools[i + 1:i + 2], fp8=True))
            caches[-1].set_kv_scales(ks, vs)
        k_out = torch.empty_like(x)
        caches[0].rope_norm_and_cache(plan, q, k_out, q, x, x, None, None, 0.0, pos, slots, n, 2)
        caches[1].reshape_and_cache(k_out, x, slots, n, 256, 256)
        torch.cuda.synchronize()
        assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3]), (ks, vs)


def test_rotate_special_values(cuda_device):
    """NaN and infinity stay in their row and pair; a zero row stays zero."""
    r = Rotate(20, 4, 2, 128, 128, norm=False, seed=4)
    clean = Rotate(20, 4, 2, 128, 128, norm=False, seed=4)
    r.q[3, 1, 5] = float("nan")
    r.q[4, 2, :] = 0
    r.run()
    clean.run()
    torch.cuda.synchronize()
    assert torch.isnan(r.q_out[3, 1, [5, 69]]).all() and int(torch.isnan(r.q_out).sum()) == 2
    assert (r.q_out[4, 2] == 0).all()
    keep = torch.ones(21, 4, 128, dtype=torch.bool, device="cuda")
    keep[3, 1, [5, 69]] = False
    keep[4, 2] = False
    assert torch.equal(r.q_out[keep], clean.q_out[keep])
    z = Rotate(2, 4, 2, 128, 128, norm=True, seed=4)
    z.q[:] = 0
    z.run()
    torch.cuda.synchronize()
    assert (z.q_out[:-1] == 0).all()


# ---- read-back ------------------------------------------------------------------------------
def f8_values(b):
    """The cache format's values of bytes: exponent 15 is infinity or NaN."""
    b = b.to(torch.int64)
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.pow(2.0, (e - 7).double()))
    v = torch.where(e == 15, torch.where(m == 0, math.inf, math.nan), v)
    return torch.where(b >= 128, -v, v)


class Gather:
    def __init__(self, lens, starts, hkv, head, block=16, fp8=False, f16=False, seed=0, extra=3, pad=0, raw=False):
        g = gen(seed)
        t = T16[f16]
        self.lens, self.starts, self.hkv, self.head, self.block, self.fp8 = lens, starts, hkv, head, block, fp8
        st = starts or [0] * len(lens)
        per = [-(-(n + s) // block) for n, s in zip(lens, st)]
        nb = sum(per) + extra
        order = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
        self.mb = max(max(per), 1) + 1
        self.tables = torch.full((len(lens), self.mb), -1, dtype=torch.int32, device="cuda")  # never to be followed
        for i, n in enumerate(per):
            self.tables[i, :n] = order[sum(per[:i]):sum(per[:i]) + n]
        x = 16 if fp8 else 8
        shapes = ((nb, hkv, head // x, block, x), (nb, hkv, head, block))
        if fp8:
            self.pools = [torch.randint(0, 256, s, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
                          for s in shapes]
        elif raw:  # every bit pattern
            self.pools = [torch.randint(-32768, 32768, s, generator=g, device="cuda").to(torch.int16).view(t)
                          for s in shapes]
        else:
            self.pools = [randn(g, *s, t=t) for s in shapes]
        self.cache = pa.PagedCache(block, nb, head, hkv, dtype=0 if f16 else 1, key_pools=self.pools[:1],
                                   value_pools=self.pools[1:], fp8=fp8)
        self.scales = (0.0371, 1.7) if fp8 else (1.0, 1.0)
        if fp8:
            self.cache.set_kv_scales(*self.scales)
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.total = int(self.cu[-1])
        self.key = torch.full((self.total + 2, hkv + pad, head), 7.0, dtype=t, device="cuda")
        self.value = torch.full((self.total + 2, hkv + pad, head), 7.0, dtype=t, device="cuda")

    def run(self, stream=0):
        row = self.key.stride(0)
        self.cache.gather(self.key, self.value, self.tables,
                          np.array(self.starts, dtype=np.int32) if self.starts else None, self.cu, len(self.lens), self.mb,
                          key_stride=row, value_stride=row, stream=stream)

    def want(self):
        ks, vs = [], []
        k, v = self.pools
        for i, n in enumerate(self.lens):
            at = (self.starts[i] if self.starts else 0) + torch.arange(n, device="cuda")
            blk, off = self.tables[i][at // self.block].long(), at % self.block
            kk, vv = k[blk, :, :, off].flatten(2), v[blk, :, :, off]
            if self.fp8:
                kk, vv = ((f8_values(b).float() * torch.tensor(s, dtype=torch.float32, device="cuda")).to(self.key.dtype)
                          for b, s in zip((kk, vv), self.scales))
            ks.append(kk)
            vs.append(vv)
        return torch.cat(ks), torch.cat(vs)

    def check(self):
        torch.cuda.synchronize()
        self.cache.check_errors()
        for got, want in zip((self.key, self.value), self.want()):
            mine = got[:self.total, :self.hkv]
            same = mine.contiguous().view(torch.int16) == want.contiguous().view(torch.int16)
            if self.fp8:
                same |= torch.isnan(mine) & torch.isnan(want)
            assert same.all()
            assert (got[self.total:] == 7.0).all() and (got[:, self.hkv:] == 7.0).all()


@pytest.mark.parametrize("head", HEADS)
def test_gather_head_sizes(cuda_device, head):
    for block in ((8, 16, 32) if head == 128 else (16, 32) if head < 128 else (16,)):
        r = Gather([1, 17, 0, 100, 33], None, 3, head, block=block, seed=head, raw=True, pad=block % 3)
        r.run()
        r.check()


@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("starts", [None, [0, 1, 7, 8, 31, 100], [16, 16, 32, 48, 64, 5]])
def test_gather_ranges(cuda_device, block, starts):
    for lens in ([1, 2, 16, 40, 1, 300], [0, 0, 5, 0, 0, 0], [700, 1, 8, 9, 2000, 31]):
        r = Gather(lens, starts, 8, 128, block=block, seed=len(lens), f16=block == 8)
        r.run()
        r.check()


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("f16", [False, True])
def test_gather_fp8_every_byte(cuda_device, block, f16):
    r = Gather([5, 64, 0, 777], [3, 0, 9, 16], 2, 128, block=block, fp8=True, f16=f16, seed=block)
    r.run()
    r.check()


def test_gather_more_sequences_than_one_launch_takes(cuda_device):
    lens = [(i * 7) % 23 for i in range(600)]
    r = Gather(lens, [(i * 5) % 17 for i in range(600)], 2, 64, seed=1)
    r.run()
    r.check()


def test_gather_bad_block_ids_are_reported_and_not_followed(cuda_device):
    r = Gather([50, 40], None, 2, 128, seed=1)
    k, v = r.want()
    r.tables[0, 1] = 10 ** 6
    r.tables[1, 2] = -5
    r.run()
    torch.cuda.synchronize()
    with pytest.raises(pa.PagedAttnError) as e:
        r.cache.check_errors()
    assert e.value.status == 4
    keep = torch.ones(90, dtype=torch.bool)
    keep[16:32] = False
    keep[50 + 32:] = False
    assert torch.equal(r.key[:90][keep], k[keep]) and torch.equal(r.value[:90][keep], v[keep])
    assert (r.key[:90][~keep] == 7.0).all() and (r.value[:90][~keep] == 7.0).all()


def test_gather_refusals(cuda_device):
    r = Gather([10, 20], None, 2, 64, seed=1)
    cu = r.cu
    for change in (dict(cu=np.array([0, 20, 10], np.int32)), dict(starts=[0, 10 ** 6]), dict(starts=[-1, 0])):
        r.cu, r.starts = change.get("cu", cu), change.get("starts")
        with pytest.raises(pa.PagedAttnError):
            r.run()
    r.cu, r.starts = cu, None
    with pytest.raises(pa.PagedAttnError):
        r.cache.gather(r.key, r.value, r.tables, None, cu, 2, r.mb, key_stride=8)
    with pytest.raises(pa.PagedAttnError):
        r.cache.gather(r.key, r.value, r.tables, None, cu, 2, r.mb, layer=1)
    r.cache.gather(r.key, r.value, r.tables, None, cu, 0, r.mb)  # nothing to do
    r.run()
    r.check()


# ---- prompt attention ---------------------------------------------------------------------------
def attend_exact(q, k, v, cu_q, cu_kv, scale, softcap=1.0):
    """(rows in 64 bits, sum p|v|) with masked keys and values never touched."""
    g = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i in range(len(cu_q) - 1):
        a, b, m, n = (int(x) for x in (cu_q[i], cu_q[i + 1], cu_kv[i], cu_kv[i + 1]))
        if a == b or m == n:
            continue
        limit = torch.arange(n - m - (b - a), n - m, device=q.device)
        sees = torch.arange(n - m, device=q.device)[None] <= limit[:, None]
        kk = k[m:n].double().repeat_interleave(g, 1).transpose(0, 1)
        vv = v[m:n].double().repeat_interleave(g, 1).transpose(0, 1)
        x = q[a:b].double().transpose(0, 1) @ kk.transpose(1, 2) * scale
        if softcap != 1.0:
            x = torch.tanh(x / softcap) * softcap
        x = x.masked_fill(~sees, -math.inf)
        p = torch.softmax(x, -1).masked_fill(~sees.any(-1)[:, None], 0.0)
        out[a:b] = (p @ vv).transpose(0, 1)
        mag[a:b] = (p @ vv.abs()).transpose(0, 1)
    return out, mag


def attend_bound(t, ref, mag, kv_max, v_max=8.0):
    u = half_step(t)
    b = (u + 2.0 ** -13) * (mag + ref.abs())
    return b + (kv_max * 2.0 ** -25 * v_max + 2.0 ** -24 if t == torch.float16 else 2.0 ** -120)


class Attend:
    def __init__(self, q_lens, kv_lens, hq, hkv, head, f16=False, seed=0, softcap=1.0, scale=None, qk=1.4, pad=0, first=0):
        g = gen(seed)
        t = T16[f16]
        self.hq, self.hkv, self.head, self.softcap = hq, hkv, head, softcap
        self.scale = head ** -0.5 if scale is None else scale
        self.cu_q = (first + np.concatenate([[0], np.cumsum(q_lens)])).astype(np.int32)
        self.cu_kv = np.concatenate([[0], np.cumsum(kv_lens)]).astype(np.int32)
        nq, nk = int(self.cu_q[-1]), int(self.cu_kv[-1])
        self.q = randn(g, nq, hq + pad, head, t=t, scale=qk)
        self.k = randn(g, nk, hkv + pad, head, t=t, scale=qk)
        self.v = randn(g, nk, hkv + 2 * pad, head, t=t)
        self.out = torch.full((nq + 3, hq + pad, head), 7.0, dtype=t, device="cuda")
        self.first, self.n = first, len(q_lens)
        self.cache = pa.PagedCache(16, 2, head, hkv, dtype=0 if f16 else 1)
        self.bytes = self.cache.prompt_workspace_bytes()
        self.ws = torch.full((self.bytes // 2,), 0x7FFF, dtype=torch.int16, device="cuda")  # NaN patterns

    def run(self, stream=0, out=None, same=False):
        out = self.out if out is None else out
        self.cache.prompt_attention(out, self.q, self.k, self.v, self.cu_q, None if same else self.cu_kv, self.n, self.hq,
                                    self.scale, self.ws, self.bytes, softcap=self.softcap, q_stride=self.q.stride(0),
                                    k_stride=self.k.stride(0), v_stride=self.v.stride(0), out_stride=out.stride(0),
                                    stream=stream)

    def check(self):
        torch.cuda.synchronize()
        self.cache.check_errors()
        nq = int(self.cu_q[-1])
        ref, mag = attend_exact(self.q[:, :self.hq], self.k[:, :self.hkv], self.v[:, :self.hkv], self.cu_q, self.cu_kv,
                                self.scale, self.softcap)
        kv_max = int(np.diff(self.cu_kv).max()) if self.n else 0
        got = self.out[self.first:nq, :self.hq]
        bound = attend_bound(got.dtype, ref, mag, kv_max)[self.first:]
        off = (got.double() - ref[self.first:]).abs()
        assert torch.isfinite(got).all()
        worst = (off / bound).max().item() if off.numel() else 0.0
        assert worst <= 1.0, f"{int((off > bound).sum())} of {off.numel()} elements beyond the bound, worst {worst:.2f} of it"
        assert (self.out[nq:] == 7.0).all() and (self.out[:, self.hq:] == 7.0).all() and (self.out[:self.first] == 7.0).all()
        return worst


@pytest.mark.parametrize("head", HEADS)
@pytest.mark.parametrize("f16", [False, True])
def test_attend_head_sizes(cuda_device, head, f16):
    for hq, hkv in ((4, 4), (8, 2), (14, 2)):
        r = Attend([1, 130, 70, 300], [1, 130, 200, 300], hq, hkv, head, f16=f16, seed=head)
        r.run()
        r.check()


@pytest.mark.parametrize("group", [1, 2, 3, 5, 6, 7, 8, 12, 24, 33, 64, 100, 128])
def test_attend_group_sizes(cuda_device, group):
    r = Attend([3, 257, 40], [150, 257, 41], 2 * group, 2, 128, seed=group)
    r.run()
    r.check()
    r = Attend([5, 60], [5, 333], group, 1, 256, seed=group, f16=True)
    r.run()
    r.check()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000])
def test_attend_lengths(cuda_device, n):
    for head in (64, 128, 192):
        r = Attend([n], [n], 8, 2, head, seed=n)
        r.run(same=True)
        r.check()
        r = Attend([n, 1, n], [n + 129, n, 2 * n + 1], 4, 2, head, seed=n)
        r.run()
        r.check()


def test_attend_rows_without_keys(cuda_device):
    """Queries before the first key, sequences without keys or without queries."""
    for head in (64, 128, 256):
        r = Attend([300, 5, 0, 77, 130, 0], [170, 0, 9, 78, 1, 0], 8, 2, head, seed=1, first=4)
        r.run()
        r.check()
        assert (r.out[4:4 + 130, :8] == 0).all() and (r.out[304:309, :8] == 0).all()
    r = Attend([4, 2], [0, 0], 4, 2, 128)
    r.cu_kv += 11  # no key anywhere, and no buffer of keys
    r.k, r.v = torch.empty(0, 2, 128, dtype=r.k.dtype, device="cuda"), torch.empty(0, 2, 128, dtype=r.k.dtype, device="cuda")
    r.run()
    torch.cuda.synchronize()
    assert (r.out[:6] == 0).all() and (r.out[6:] == 7.0).all()


@pytest.mark.parametrize("head", [64, 128, 192])
def test_attend_few_rows_over_long_keys(cuda_device, head):
    for q, kv, hq, hkv in (([1], [20000], 8, 1), ([1, 5, 2], [9000, 12345, 300], 32, 8), ([16], [16384], 4, 4)):
        r = Attend(q, kv, hq, hkv, head, seed=2)
        r.run()
        r.check()


def test_attend_long_prompt(cuda_device):
    r = Attend([4500], [4500], 8, 2, 128, seed=3)
    r.run()
    r.check()
    r = Attend([900, 1100], [5000, 6100], 16, 4, 128, seed=4, f16=True)
    r.run()
    r.check()


def test_attend_many_sequences(cuda_device):
    """More sequences than one launch takes."""
    rng = np.random.default_rng(0)
    q = rng.integers(0, 9, 700).tolist()
    kv = [n + int(m) for n, m in zip(q, rng.integers(0, 300, 700))]
    r = Attend(q, kv, 8, 2, 64, seed=5)
    r.run()
    r.check()


@pytest.mark.parametrize("softcap", [1.0, 20.0])
@pytest.mark.parametrize("qk", [0.01, 4.0])
def test_attend_logit_ranges(cuda_device, softcap, qk):
    """Nearly uniform and nearly one-hot weights; rising logits that move the maximum often."""
    r = Attend([200, 700], [200, 1500], 8, 2, 128, seed=6, softcap=softcap, qk=qk)
    r.run()
    r.check()
    r = Attend([150], [3000], 4, 1, 64, seed=7, softcap=softcap, qk=1.0)
    r.k *= torch.linspace(0.1, 12, 3000, device="cuda")[:, None, None].to(r.k.dtype)
    r.run()
    r.check()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("head", [64, 128, 192])
@pytest.mark.parametrize("spikes", [[70], [130], [200], [130, 255], [140, 200, 300, 390], [511], [383, 640, 1022]])
@pytest.mark.parametrize("height", [60.0, 160.0])
def test_attend_sudden_maxima(cuda_device, f16, head, spikes, height):
    """Keys whose logits lie tens of powers of two above everything before them - or more than fp32's
    exponent - in either half of a key tile or in both, in the first, a middle and the last tile, for
    some rows and not for others."""
    for q, kv in (([60], [1024]), ([300], [300]), ([700, 33], [1024, 1024])):
        r = Attend(q, kv, 8, 2, head, f16=f16, seed=sum(spikes), qk=0.7)
        sign = torch.where(torch.rand(r.q.shape[:2], generator=gen(5), device="cuda") < 0.6, 8.0, -8.0)
        r.q[..., 0] = sign.to(r.q.dtype)
        r.k[..., 0] = 0
        for n, j in enumerate(spikes):
            for base in r.cu_kv[:-1]:
                if base + j < int(r.cu_kv[-1]):
                    r.k[base + j, :, 0] = (height + 40.0 * n) * head ** 0.5 / 8
        r.run()
        r.check()


def test_attend_strides(cuda_device):
    r = Attend([33, 200], [133, 300], 8, 2, 96, seed=8, pad=3, first=2)
    r.run()
    r.check()


def test_attend_masked_places_do_not_reach(cuda_device):
    """NaN, infinity and the type's largest numbers in keys and values that a row does not see:
    later tokens of its own sequence and everything of the others."""
    for head, hq, hkv in ((64, 8, 2), (128, 8, 2), (256, 4, 1)):
        for f16 in (False, True):
            q, kv = [40, 300, 7], [40, 420, 7]
            r = Attend(q, kv, hq, hkv, head, seed=head, f16=f16)
            r.run()
            torch.cuda.synchronize()
            clean = r.out.clone()
            big = torch.finfo(r.k.dtype).max
            bad = 40 + 120 + 250  # key 370 of the middle sequence: query 250 is the first that sees it
            r.k[bad] = float("nan")
            r.k[bad + 2, :, ::2] = -float("inf")
            r.v[bad, :, 3] = float("nan")
            r.v[bad + 1] = float("inf")
            r.v[bad + 2, :, 5] = -float("inf")
            r.v[bad + 3] = big
            r.k[460:] = float("nan")
            r.v[460:] = float("nan")
            r.q[340:] = float("nan")
            r.run()
            torch.cuda.synchronize()
            r.cache.check_errors()
            rows = 40 + 250
            assert torch.isfinite(r.out[:rows]).all()
            ref, mag = attend_exact(r.q[:rows], r.k[:40 + 370], r.v[:40 + 370],
                                    [0, 40, rows], [0, 40, 40 + 370], r.scale)
            off = (r.out[:rows].double() - ref).abs()
            assert (off <= attend_bound(r.out.dtype, ref, mag, 420)).all()
            same = (r.out[:rows] == clean[:rows]).flatten(1).all(1)
            assert same[:40].all(), "another sequence's values reached the first one"
            assert torch.isnan(r.out[rows:347]).any(-1).all(), "a row that sees a NaN key has to show it"


@pytest.mark.parametrize("f16", [False, True])
def test_attend_masked_places_of_a_cut_item(cuda_device, f16):
    """The same where the item is cut over many CTAs and rows are put right by the join, and where it
    is one query tile on two places."""
    for q, kv, hq, hkv in ((3, 9000, 8, 1), (40, 6000, 4, 1), (100, 3000, 8, 2)):
        r = Attend([q, 2], [kv, 50], hq, hkv, 128, seed=q, f16=f16)
        r.run()
        torch.cuda.synchronize()
        clean = r.out.clone()
        r.v[kv - 1, :, 3] = float("nan")   # the last query alone sees it
        r.v[kv - 2] = float("inf")         # the last two
        r.v[kv + 10:] = float("nan")       # the other sequence
        r.run()
        torch.cuda.synchronize()
        r.cache.check_errors()
        got = r.out[:q - 2]
        ref, mag = attend_exact(r.q[:q - 2], r.k[:kv - 2], r.v[:kv - 2], [0, q - 2], [0, kv - 2], r.scale)
        assert torch.isfinite(got).all() and ((got.double() - ref).abs() <= attend_bound(got.dtype, ref, mag, kv)).all()
        assert (r.out[q - 2, :, :] == float("inf")).all() and torch.isnan(r.out[q - 1, :, 3]).all()
        assert (r.out[q - 1, :, 4:] == float("inf")).all()
        same = (got == clean[:q - 2]) | ((got.double() - clean[:q - 2].double()).abs() <= attend_bound(got.dtype, ref, mag, kv))
        assert same.all()


def test_attend_special_values_propagate(cuda_device):
    r = Attend([64], [64], 4, 1, 128, seed=1)
    r.q[10, 2, 0] = float("nan")
    r.v[20, 0, 4] = float("inf")
    r.run()
    torch.cuda.synchronize()
    assert torch.isnan(r.out[10, 2]).all() and torch.isfinite(r.out[10, [0, 1, 3]]).all()
    assert torch.isfinite(r.out[:20, [0, 1, 3]]).all() and (r.out[20:64, :, 4] == float("inf")).all()
    assert torch.isfinite(r.out[20:64, :, [0, 3, 5, 127]]).all()


def test_attend_same_bits_every_time(cuda_device):
    r = Attend([700, 3, 1200], [900, 5000, 1200], 16, 4, 128, seed=9)
    r.run()
    torch.cuda.synchronize()
    first = r.out.clone()
    for _ in range(5):
        r.ws.fill_(0x7FFF)
        r.out.fill_(7.0)
        r.run()
    torch.cuda.synchronize()
    assert torch.equal(first, r.out)


def test_attend_refusals(cuda_device):
    r = Attend([10, 20], [10, 20], 4, 2, 64, seed=1)
    cu = r.cu_q
    for bad in ([0, 20, 10], [-1, 5, 10]):
        r.cu_q = np.array(bad, np.int32)
        with pytest.raises(pa.PagedAttnError):
            r.run()
    r.cu_q = cu
    r.scale, ok = 0.0, r.scale
    with pytest.raises(pa.PagedAttnError):
        r.run()
    r.scale = ok
    r.bytes -= 1
    with pytest.raises(pa.PagedAttnError):
        r.run()
    r.bytes += 1
    r.hq = 3
    with pytest.raises(pa.PagedAttnError):
        r.run()
    r.hq = 4
    r.cache.prompt_attention(r.out, r.q, r.k, r.v, cu, None, 0, 4, 0.1, r.ws, r.bytes)
    torch.cuda.synchronize()
    assert (r.out == 7.0).all()
    r.run()
    r.check()


# ---- streams, graphs, large offsets ------------------------------------------------------------
def test_other_stream_and_captured_graph(cuda_device):
    """All three calls on a stream of their own, then captured and replayed on new inputs."""
    s = torch.cuda.Stream()
    rot, gat, att = Rotate(70, 8, 2, 128, 128, seed=1), Gather([100, 9], [4, 0], 2, 128, seed=2), \
        Attend([70, 3], [170, 900], 8, 2, 128, seed=3)
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        for r in (rot, gat, att):
            r.run(stream=s.cuda_stream)
    s.synchronize()
    for r in (rot, gat, att):
        r.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for r in (rot, gat, att):
            r.run(stream=torch.cuda.current_stream().cuda_stream)
    for seed in (11, 12):
        g = gen(seed)
        rot.qkv.copy_(randn(g, *rot.qkv.shape))
        gat.pools[0].copy_(randn(g, *gat.pools[0].shape))
        att.q.copy_(randn(g, *att.q.shape))
        att.v.copy_(randn(g, *att.v.shape))
        for r in (rot.q_out, rot.k_out, gat.key, gat.value, att.out):
            r.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        for r in (rot, gat, att):
            r.check()


def test_pool_offsets_beyond_32_bits(cuda_device):
    """A pool of 2.3 G elements: its last blocks are written and read back, its first stay."""
    nb, hkv, head, block = 140000, 8, 128, 16
    pools = [torch.zeros(nb * hkv * head * block, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache = pa.PagedCache(block, nb, head, hkv, key_pools=pools[:1], value_pools=pools[1:])
    g = gen(0)
    q, k, v = (randn(g, 50, h, head) for h in (8, hkv, hkv))
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ids = torch.tensor([nb - 1, nb - 7, nb - 3, 0], dtype=torch.int32, device="cuda")
    at = torch.arange(50, device="cuda")
    slots = ids.long()[at // 16] * 16 + at % 16
    plan = pa.RopePlan(head, 1e6)
    cache.rope_norm_and_cache(plan, q_out, k_out, q, k, v, None, None, 1e-6, at.to(torch.int32), slots, 50, 8)
    key, value = torch.empty_like(k), torch.empty_like(v)
    cache.gather(key, value, ids[None], None, np.array([0, 50], np.int32), 1, 4)
    torch.cuda.synchronize()
    cache.check_errors()
    assert torch.equal(key, k_out) and torch.equal(value, v)
    assert int(torch.count_nonzero(pools[0][hkv * head * block:-8 * hkv * head * block])) == 0


def test_row_offsets_beyond_32_bits(cuda_device):
    """Keys and queries in rows 2^23 elements apart: offsets of 2.5 G elements."""
    stride, n = 1 << 23, 300
    big = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda")
    r = Attend([n], [n], 2, 1, 64, seed=1)
    views = []
    for i, x in enumerate((r.q, r.k, r.v, r.out[:n])):
        view = big.as_strided(x.shape, (stride, 64, 1), 4096 * i)
        view.copy_(x)
        views.append(view)
    r.q, r.k, r.v = views[:3]
    r.run(out=views[3])
    torch.cuda.synchronize()
    r.out[:n] = views[3]
    r.check()


# ---- the run a serving program makes of them ----------------------------------------------------
@pytest.mark.parametrize("head,block,fp8,f16", [(128, 16, False, False), (128, 32, True, False), (64, 32, False, True),
                                                (128, 8, False, False), (256, 16, False, False)])
def test_prompt_in_two_chunks_over_a_cache(cuda_device, head, block, fp8, f16):
    """First chunk: rotated, written and attended straight from its projections.  Second chunk:
    rotated and written, the whole context read back, attended over it; then one decode token
    by the paged attention.  Each output against the 64-bit formula on the rows the calls saw,
    and the second chunk against the paged attention over the same pool."""
    t = T16[f16]
    hq, hkv, g = 8, 2, gen(head + block)
    lens = [(200, 90), (33, 1), (64, 130)]
    total = [a + b + 1 for a, b in lens]
    mb = max(-(-n // block) for n in total)
    per = [-(-n // block) for n in total]
    nb = sum(per)
    tables = torch.zeros(3, mb, dtype=torch.int32, device="cuda")
    order = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    for i, n in enumerate(per):
        tables[i, :n] = order[sum(per[:i]):sum(per[:i]) + n]
    cache = pa.PagedCache(block, nb, head, hkv, dtype=0 if f16 else 1, fp8=fp8)
    if fp8:
        cache.set_kv_scales(1 / 16, 1 / 32)
    plan = pa.RopePlan(head, 1e6, scaling="yarn", factor=4.0, original_max_position=4096)
    w = (1 + 0.1 * torch.randn(head, generator=g, device="cuda")).to(t)
    ws_n, pws_n = cache.prompt_workspace_bytes(), cache.workspace_bytes()
    ws = torch.empty(ws_n, dtype=torch.uint8, device="cuda")
    pws = torch.empty(pws_n, dtype=torch.uint8, device="cuda")
    scale = head ** -0.5

    def project(first, count):
        """Rotated queries, keys and the values of `count[i]` tokens from first[i] on, in the cache."""
        pos = torch.cat([torch.arange(f, f + n) for f, n in zip(first, count)]).to("cuda")
        seq = torch.repeat_interleave(torch.arange(3), torch.tensor(count)).to("cuda")
        n = len(pos)
        slots = tables[seq, pos // block].long() * block + pos % block
        q, k, v = randn(g, n, hq, head, t=t), randn(g, n, hkv, head, t=t), randn(g, n, hkv, head, t=t)
        k_out = torch.empty_like(k)
        cache.rope_norm_and_cache(plan, q, k_out, q, k, v, w, w, 1e-6, pos.to(torch.int32), slots, n, hq)
        return q, k_out, v

    def cu(x):
        return np.concatenate([[0], np.cumsum(x)]).astype(np.int32)

    def hold(out, q, k, v, cq, ck):
        ref, mag = attend_exact(q, k, v, cq, ck, scale)
        assert ((out.double() - ref).abs() <= attend_bound(t, ref, mag, max(total))).all()

    a, b = [x for x, _ in lens], [y for _, y in lens]
    q, k, v = project([0] * 3, a)
    out = torch.empty_like(q)
    cache.prompt_attention(out, q, k, v, cu(a), None, 3, hq, scale, ws, ws_n)
    hold(out, q, k, v, cu(a), cu(a))

    q, k, v = project(a, b)
    both = [x + y for x, y in lens]
    key = torch.empty(sum(both), hkv, head, dtype=t, device="cuda")
    value = torch.empty_like(key)
    cache.gather(key, value, tables, None, cu(both), 3, mb)
    out = torch.empty_like(q)
    cache.prompt_attention(out, q, key, value, cu(b), cu(both), 3, hq, scale, ws, ws_n)
    torch.cuda.synchronize()
    cache.check_errors()
    hold(out, q, key, value, cu(b), cu(both))
    if not fp8:  # the second chunk's own rows come back as they were written
        at = np.concatenate([np.arange(cu(both)[i] + a[i], cu(both)[i + 1]) for i in range(3)])
        assert torch.equal(key[at], k) and torch.equal(value[at], v)
    paged = torch.empty_like(q)
    ctx = torch.tensor(both, dtype=torch.int32, device="cuda")
    cache.varlen(paged, q, tables, ctx, cu(b), 3, hq, mb, scale, pws, pws_n, context_lens_host=np.array(both, np.int32))
    torch.cuda.synchronize()
    ref, mag = attend_exact(q, key, value, cu(b), cu(both), scale)
    # two results that each keep the bound (an FP8 pool's read-back rounds its values once more)
    assert ((out.double() - paged.double()).abs() <= 3 * attend_bound(t, ref, mag, max(total)) + 1e-2 * ref.abs().mean()).all()

    q, k, v = project(both, [1] * 3)
    paged, out = torch.empty_like(q), torch.empty_like(q)
    cache.decode(paged, q, tables, ctx + 1, 3, hq, mb, scale, pws, pws_n)
    key = torch.empty(sum(total), hkv, head, dtype=t, device="cuda")
    value = torch.empty_like(key)
    cache.gather(key, value, tables, None, cu(total), 3, mb)
    cache.prompt_attention(out, q, key, value, cu([1] * 3), cu(total), 3, hq, scale, ws, ws_n)
    torch.cuda.synchronize()
    cache.check_errors()
    hold(out, q, key, value, cu([1] * 3), cu(total))
    ref, mag = attend_exact(q, key, value, cu([1] * 3), cu(total), scale)
    assert ((out.double() - paged.double()).abs() <= 3 * attend_bound(t, ref, mag, max(total)) + 1e-2 * ref.abs().mean()).all()


def test_launches_are_counted(cuda_device):
    before = pa.kernel_launch_count()
    Rotate(3, 4, 2, 64, 64).run()
    Gather([5], None, 2, 64).run()
    Attend([3], [3], 4, 2, 64).run()
    torch.cuda.synchronize()
    assert pa.kernel_launch_count() >= before + 3
