"""GPU tests of pa_prompt_attention where logits jump by about as much as fp32's exponent holds.

A tile's probabilities are taken against a reference that the tiles before it set.  In bf16 they
and their sum may then reach fp32's largest numbers: 88.7 nats above the reference is 2^128.
Heights here are in nats above the other logits; the tolerance is attend_bound of
test_gpu_prompt_path, whose 2^-13 covers what logits of this size add: a dot product's rounding and
that of logit - reference (2^-17 for numbers around 128), a logarithm's and its exponential's
(the same again), and a reciprocal below 2^-126, which keeps 22 bits.
"""
import pytest
import torch

from test_gpu_prompt_path import Attend, attend_bound, gen

pytestmark = pytest.mark.gpu

# (query lengths, key lengths): one query tile on two places, two query tiles, both of three key tiles
# and never cut; then items that are cut, and many of which some are
SHAPES = {
    "places": ([20], [384]),
    "tiles": ([64], [384]),
    "cut": ([20], [1024]),
    "cut-tiles": ([64], [1024]),
    "many": ([20] * 90, [512] * 90),
    "prompt": ([700, 33], [1024, 1024]),
}


def raised(shape, head, heights, f16=False, v_scale=0.1, seed=0):
    """Attend over `shape` with key j of every sequence `heights(j, kv_len, seq)` nats above the rest."""
    q, kv = SHAPES[shape]
    r = Attend(q, kv, 8, 2, head, f16=f16, seed=seed, qk=0.2)
    r.v = (r.v.float() * v_scale).to(r.v.dtype)
    r.q[..., :2] = 8.0
    r.k[..., :2] = 0.0
    unit = head ** 0.5 / 8
    for s, base in enumerate(r.cu_kv[:-1]):
        for j, height in heights(kv[s], s):
            x = torch.tensor(height * unit)
            hi = x.to(r.k.dtype)  # in two elements, so that a height is met to a few thousandths
            r.k[int(base) + j, :, 0] = hi
            r.k[int(base) + j, :, 1] = (x - hi.float()).to(r.k.dtype)
    return r


def spread(tile, n):
    """n keys over both halves of a key tile."""
    return [tile * 128 + i * 128 // n for i in range(n)]


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("head", [64, 128, 192])
@pytest.mark.parametrize("n", [2, 16, 128])
def test_sums_around_the_largest_number(cuda_device, shape, head, n):
    """Several equal keys whose probabilities, or only their sum, leave fp32 - in the last key tile, in the one
    before it, and in the second one."""
    for height in (83.0, 84.6, 85.3, 86.0, 87.2, 88.0, 88.4, 88.6, 89.0):
        for tile in (-1, -2, 1):
            r = raised(shape, head, lambda kv, s: [(j, height) for j in spread(tile % (kv // 128), n)])
            r.run()
            r.check()


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("head", [64, 128, 192])
def test_one_half_of_the_columns_overflows(cuda_device, shape, head):
    """Values that take one half of a row's outputs beyond fp32 in the last key tile and leave the other there."""
    for height in (70.0, 84.6, 88.4):
        r = raised(shape, head, lambda kv, s: [(j, height) for j in spread(kv // 128 - 1, 16)])
        r.v[..., :head // 2] = (r.v[..., :head // 2].float() * 2.0 ** 40).to(r.v.dtype)
        r.run()
        r.check()


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("head", [64, 128, 192])
@pytest.mark.parametrize("f16", [False, True])
def test_parts_with_references_far_apart(cuda_device, shape, head, f16):
    """Key tiles of any height: the pieces and places of an item end with references up to fp32's exponent range
    and more apart, while the sums of those left behind make up for it."""
    heights = (0.0, 60.0, 80.0, 86.0, 87.0, 87.5, 88.0, 89.0, 91.0, 120.0, 176.0)
    for seed in range(12):
        pick = torch.randint(0, len(heights), (128, 64), generator=torch.Generator().manual_seed(seed)).tolist()

        def tiles(kv, s):
            return [(j, heights[pick[s][t]]) for t in range(1, kv // 128) for j in spread(t, 1 + pick[s][63 - t] % 3)]
        r = raised(shape, head, tiles, f16=f16, seed=seed)
        r.run()
        r.check()


@pytest.mark.parametrize("head", [64, 128])
def test_two_places_far_apart(cuda_device, head):
    """Tiles 0 and 2 share a place, tile 1 has its own: the sum of the first, 2^125 against a reference of 0,
    next to a reference of 2^127."""
    for low, high in ((87.0, 88.0), (88.4, 90.0), (86.0, 89.0)):
        r = raised("places", head, lambda kv, s: [(200, high), (260, low)])
        r.run()
        r.check()


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("log2_v", [40, 90, 100])
def test_large_values_behind_a_jump(cuda_device, shape, log2_v):
    """bf16 values of up to 2^100: probabilities far above 1 would take the weighted sum beyond fp32 although the
    result is inside."""
    for height in (15.0, 30.0, 45.0):
        for tile in (-1, 1):
            r = raised(shape, 128, lambda kv, s: [(j, height) for j in spread(tile % (kv // 128), 2)],
                       v_scale=2.0 ** log2_v)
            r.run()
            r.check()


def test_a_recomputed_row_outlasts_a_wait(cuda_device):
    """One row over two million keys jumps beyond fp32's exponent: recomputing it takes longer than the second that
    the CTA's other warps wait for anything, which is no error while it gets on.  160 query tiles, so that the
    row's item is not cut."""
    n, head, queries = 1 << 21, 256, 160 * 128
    r = Attend([queries], [128], 1, 1, head)
    g = gen(1)
    r.cu_kv[1] = n
    r.k, r.v = (torch.empty(n, 1, head, dtype=r.q.dtype, device="cuda").normal_(0, s, generator=g) for s in (0.7, 1.0))
    r.q[..., 0], r.k[..., 0] = 0.0, 0.0
    r.q[0, 0, 0], r.k[n // 2, 0, 0] = 8.0, 100.0 * head ** 0.5 / 8
    r.run()
    torch.cuda.synchronize()
    r.cache.check_errors()
    seen = n - queries + 1
    parts = [slice(i, min(i + (1 << 18), seen)) for i in range(0, seen, 1 << 18)]
    p = torch.softmax(torch.cat([r.k[s, 0].double() @ r.q[0, 0].double() for s in parts]) * r.scale, 0)
    ref = sum(p[s] @ r.v[s, 0].double() for s in parts)
    mag = sum(p[s] @ r.v[s, 0].double().abs() for s in parts)
    assert ((r.out[0, 0].double() - ref).abs() <= attend_bound(r.q.dtype, ref, mag, n)).all()
    assert torch.isfinite(r.out[:queries]).all()
