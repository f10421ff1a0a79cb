"""How exact the attention of drafted tokens is: bounds from the roundings that it may make, tight enough that a term less in a query or in a weight shows."""
import pytest

from test_gpu_attn_tree import HD, make
from test_gpu_draft import chain, dev, ints, trees

pytestmark = pytest.mark.gpu
TILES = [(1, 4, 1), (6, 20, 5), (8, 4, 1), (33, 4, 2), (60, 8, 2)]  # nodes, heads, KV heads: 4, 24, 32 rows of a tile of 16 or 32, 66 and 240 rows of 128


def in_64_bits(q, k, v, pos, parents, counts, scale=HD ** -0.5):
    """(values, sum of |weight * value|, the largest sum of a score's |products|); zeros where nothing is computed."""
    import torch
    b, t, nh, _ = q.shape
    share = nh // k.shape[1]
    want, wide, size = (torch.zeros(q.shape, device="cuda", dtype=torch.float64) for _ in range(3))
    for i in range(b):
        n, p = int(counts[i]), int(pos[i])
        seen = torch.zeros(n, p + n, dtype=torch.bool)
        seen[:, :p] = True
        for node in range(n):
            seen[node, [p + a for a in chain(parents[i], node)]] = True
        seen = seen.cuda()
        for h in range(nh):
            kk, vv, qq = k[i, h // share, :p + n].double(), v[i, h // share, :p + n].double(), q[i, :n, h].double()
            w = torch.softmax((qq @ kk.T * scale).masked_fill(~seen, -torch.inf), -1)
            want[i, :n, h], wide[i, :n, h] = w @ vv, w @ vv.abs()
            size[i, :n, h] = (qq.abs() @ kk.abs().T * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    return want, wide, size


@pytest.mark.parametrize("t,nh,kvh", TILES)
@pytest.mark.parametrize("length,spread", [(4, 1.5), (4, 6.0), (300, 6.0), (300, 0.1), (5000, 1.5), (20000, 6.0)])
def test_bf16_results_are_off_by_their_own_rounding(ctx, t, nh, kvh, length, spread):
    """Weights of few heavy keys whose values cancel, and of many light ones."""
    import torch
    from lemonade_burn_b200 import ops
    args = make(1, t, nh, kvh, [length], torch.bfloat16, seed=length, spread=spread)
    got = ops.attn_tree(*args[:3], *dev(*args[3:])).double()
    ctx.check_device_error()
    want, wide, size = in_64_bits(*args)
    # The result is rounded: 2^-8 of it. In front of that, of `wide`: a score is eight sums of 16 exact products, each cut off at 2^-22 of them, and three roundings: 2^-18 of
    # its products' size, in the weight and in the weights' sum; a weight in two terms 2^-16 and its exponential 2^-22; its sums over the keys, one in 16 keys and
    # term cut off at 2^-22, and over the weights n 2^-24; 148 parts joined 2^-16.
    slack = 2.0 ** -8 * want.abs() + 1.01 * wide * (2.0 ** -17 * size + 2.0 ** -16 + 2.0 ** -16 + 2.0 ** -21 + (length + t) * (2.0 ** -25 + 2.0 ** -24))
    off = (got - want).abs()
    assert bool((off <= slack).all()), f"off by {float((off / slack).max())} of what is allowed"


@pytest.mark.parametrize("t,nh,kvh", TILES)
@pytest.mark.parametrize("length", [3, 400])
def test_f32_queries_are_whole(ctx, t, nh, kvh, length):
    """Scores that are small differences of large products."""
    import torch
    from lemonade_burn_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(t + length)
    rand = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    q = torch.zeros(1, t, nh, HD, device="cuda")
    q[..., 0] = 1 + rand(1, t, nh)
    q[..., 1] = q[..., 0] + rand(1, t, nh) / 32
    k = torch.zeros(1, kvh, length + t, HD, device="cuda", dtype=torch.bfloat16)
    sign = torch.where(rand(1, kvh, length + t) < 0.5, -1.0, 1.0)
    k[..., 0] = (256 * sign * (1 + rand(1, kvh, length + t))).to(torch.bfloat16)
    # values of the key's sign: what a query's missing bits do to the scores is of that sign, too, and does not average out
    v = ((1 + rand(*k.shape)) * sign[..., None]).to(torch.bfloat16)
    # the second product takes most of the first one away
    k[..., 1] = (-k[..., 0].float() + 40 * (rand(1, kvh, length + t) - 0.5)).to(torch.bfloat16)
    args = q, k, v, ints([length]), trees(1, t, t), ints([t])
    got = ops.attn_tree(q, k, v, *dev(*args[3:])).double()
    ctx.check_device_error()
    want, wide, size = in_64_bits(*args)
    # Three products of two dimensions each come to a score: a sum is cut off at 2^-23 of its largest addend for each of three, two more are rounded, so 2^-21
    # of the products' size, twice for a weight and the weights' sum. The other roundings, of a score that is no larger than its products, an exponential, weights and
    # their sums, are below 2^-18 for 400 keys. A query in two terms is off by up to 2^-16, some 2^-18 as a rule, of each product.
    off, slack = (got - want).abs(), wide * (2.0 ** -20 * size + 2.0 ** -18)
    assert bool((off <= slack).all()), f"off by {float((off / slack).max())} of what is allowed"


@pytest.mark.parametrize("t,nh,kvh", TILES)
def test_f32_weights_are_whole(ctx, t, nh, kvh):
    """Two keys, the heavier with values of zero: a result is one weight times a value."""
    import torch
    from lemonade_burn_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(t)
    for _ in range(4):
        rand = lambda *shape: torch.rand(shape, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
        q = torch.zeros(1, t, nh, HD, device="cuda")
        q[..., 0] = (1 + rand(1, t, nh)).float()                  # one term
        k, v = torch.zeros(1, kvh, 1 + t, HD, device="cuda", dtype=torch.bfloat16), torch.zeros(1, kvh, 1 + t, HD, device="cuda", dtype=torch.bfloat16)
        k[..., 0, 0] = 6.0                                        # scores of up to 1.06
        k[..., 1:, 0] = 6.0 * rand(1, kvh, t)
        v[..., 1:, :] = 1 + rand(1, kvh, t, HD)
        args = q, k, v, ints([1]), torch.full((1, t), -1, dtype=torch.int32), ints([t])
        got = ops.attn_tree(q, k, v, *dev(*args[3:])).double()
        want, _, _ = in_64_bits(*args)
        # In steps of 2^-24. Scores: the factor 2.5, two products 1.1 each: 5 of a score's difference and of the scores, at most 1.1 each; exponential 4; in three
        # terms 1; sums of three products 6. The weights' sum: its smaller part's 10, and 1; the quotient and the product 3. A weight in two terms is off by up to 256.
        assert bool(((got - want).abs() <= 32 * 2.0 ** -24 * want.abs()).all()), float(((got - want) / want).abs().max() * 2.0 ** 24)
    ctx.check_device_error()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kvh,length", [(148, 200), (74, 470), (1, 37000)])
def test_values_that_come_late(ctx, dtype, kvh, length):
    """Walks whose last block holds the nodes and rows that nobody has written, right behind one that holds none, while something else takes the memory's bandwidth: values are
    looked at when they have landed, not when the ones in front of them in their place have."""
    import torch
    from lemonade_burn_b200 import ops
    t = 40 if kvh > 1 else 70
    q, k, v, pos, parents, counts = make(1, t, kvh if kvh > 1 else 4, kvh, [length], getattr(torch, dtype), room=90)
    on = dev(pos, parents, counts)
    first = ops.attn_tree(q, k, v, *on)
    want, wide, _ = in_64_bits(q, k, v, pos, parents, counts)
    assert bool(((first.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * wide).all())
    big = [torch.empty(1 << 28, dtype=torch.uint8, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    for i in range(40):
        with torch.cuda.stream(side):
            big[i & 1].copy_(big[1 - (i & 1)])
        assert torch.equal(ops.attn_tree(q, k, v, *on), first)
        torch.cuda.synchronize()
    ctx.check_device_error()
