"""GPU tests of the flag that pa_rope_norm_and_cache raises when a byte with exponent field 15
(infinity or NaN) goes into an FP8 cache: a cache that starts on the fast decode, which reads such
a byte as a finite number, switches to the exact one by itself.

Magnitudes that encode to such a byte, after the division by the layer's scale: 248 (halfway between 240
and 256, to even), anything to 256, 16384 and more, infinity; NaN.  From 256 to below 16384 the format
keeps three bits of a shifted mantissa, a finite byte.
"""
import pytest
import torch

import paged_attn_b200 as pa
from test_gpu_prompt_path import Rotate

pytestmark = pytest.mark.gpu

ELEMENT = 101  # beyond the 64 that rotate: a key's element arrives as it went in
SCALED = (248.0, -252.0, 16384.0, -20480.0, float("inf"), float("nan"))


class Step:
    """16 tokens into one block of a fresh FP8 cache on the fast decode, then one query over them."""

    def __init__(self, f16, seed):
        self.r = r = Rotate(16, 2, 1, 128, 64, norm=False, fp8=True, f16=f16, seed=seed)
        self.scales = (1 / 16, 1 / 8)
        r.q[0, :, ELEMENT] = 1.0
        r.cache.fp8_set_exact_decode(False)

    def put(self, which, token, scaled):
        (self.r.k if which == 0 else self.r.v)[token, 0, ELEMENT] = scaled * self.scales[which]

    def byte(self, which, token):
        blk, off = int(self.r.slots[0]) // 16, token
        if which == 0:
            return self.r.pools[0][blk, 0, ELEMENT // 16, off, ELEMENT % 16].item()
        return self.r.pools[1][blk, 0, ELEMENT, off].item()

    def attend(self, cache=None):
        r, cache = self.r, cache or self.r.cache
        tables = torch.tensor([[int(r.slots[0]) // 16]], dtype=torch.int32, device="cuda")
        lens = torch.tensor([16], dtype=torch.int32, device="cuda")
        out = torch.zeros(1, 2, 128, dtype=r.q_out.dtype, device="cuda")
        n = cache.workspace_bytes()
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        cache.decode(out, r.q_out, tables, lens, 1, 2, 1, 0.05, ws, n)
        torch.cuda.synchronize()
        cache.check_errors()
        return out[0]

    def fast(self):
        """The same pools behind a handle whose flag nothing raises."""
        c = pa.PagedCache(16, self.r.pools[0].shape[0], 128, 1, dtype=0 if self.r.q.dtype == torch.float16 else 1,
                          key_pools=self.r.pools[:1], value_pools=self.r.pools[1:], fp8=True)
        c.set_kv_scales(*self.scales)
        c.fp8_set_exact_decode(False)
        return c


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("scaled", SCALED)
def test_exponent_15_switches_the_cache_to_exact(cuda_device, f16, which, scaled):
    s = Step(f16, seed=2)
    s.put(which, 3, scaled)
    s.r.run()
    torch.cuda.synchronize()
    assert s.byte(which, 3) & 0x78 == 0x78
    out = s.attend()
    if which == 0:  # a logit that is infinite or NaN
        assert scaled < 0 or not torch.isfinite(out).any()
        if scaled < 0:  # minus infinity: as if the token were not there
            assert torch.isfinite(out).all()
            assert not torch.equal(out, s.attend(s.fast()))
    else:
        assert not torch.isfinite(out[:, ELEMENT]).any()
    if scaled > 0 or which == 1:
        assert torch.isfinite(s.attend(s.fast())).all(), "the fast decode shows the byte too: nothing was tested"


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("which", [0, 1])
def test_finite_bytes_and_skipped_slots_leave_the_flag(cuda_device, f16, which):
    """247 is 240, 300 keeps three bits of its mantissa; a token without a slot writes nothing."""
    s = Step(f16, seed=3)
    for token, scaled in ((3, 247.0), (5, 300.0), (7, -8000.0)):
        s.put(which, token, scaled)
    s.put(which, 9, float("inf"))
    for p in s.r.pools:
        p.zero_()
    s.r.slots[9] = -1
    s.r.run()
    torch.cuda.synchronize()
    assert all(s.byte(which, t) & 0x78 != 0x78 for t in range(16)) and s.byte(which, 9) == 0
    # a byte put there by hand shows which decode is in use
    blk = int(s.r.slots[0]) // 16
    s.r.pools[1][blk, 0, 33, 11] = 0x78
    assert torch.isfinite(s.attend()).all()
    s.r.cache.fp8_set_exact_decode(True)
    assert not torch.isfinite(s.attend()[:, 33]).any()
