"""Attention of drafted tokens against plain sums in 64 bits: head layouts, lengths from nothing to long, ragged batches, trees of
every shape, both types, values that are no numbers where a row does not look, strides, refusals."""
import math

import pytest

from test_gpu_draft import chain, dev, ints, trees

pytestmark = pytest.mark.gpu
HD = 128


def make(b, t, nh, kvh, lengths, dtype, shape="random", counts=None, seed=0, room=5, spread=1.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * t + b)
    cap = max(lengths) + t + room
    q = (spread * torch.randn(b, t, nh, HD, generator=g, device="cuda")).to(dtype)
    k, v = (torch.randn(b, kvh, cap, HD, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    counts = [t] * b if counts is None else counts
    for i in range(b):  # nobody has written these
        k[i, :, lengths[i] + counts[i]:], v[i, :, lengths[i] + counts[i]:] = math.nan, math.nan
    return q, k, v, ints(lengths), trees(b, t, seed, shape), ints(counts)


def expected(q, k, v, pos, parents, counts, scale=HD ** -0.5):
    """(values, the most an output may be off by) in 64 bits; NaN where nothing is computed."""
    import torch
    b, t, nh, _ = q.shape
    share = nh // k.shape[1]
    want = torch.full(q.shape, math.nan, device="cuda", dtype=torch.float64)
    slack = want.clone()
    for i in range(b):
        n, p = int(counts[i]), int(pos[i])
        if not n:
            continue
        seen = torch.zeros(n, p + n, dtype=torch.bool)
        seen[:, :p] = True
        for node in range(n):
            seen[node, [p + a for a in chain(parents[i], node)]] = True
        seen = seen.cuda()
        for h in range(nh):
            kk, vv, qq = k[i, h // share, :p + n].double(), v[i, h // share, :p + n].double(), q[i, :n, h].double()
            w = torch.softmax((qq @ kk.T * scale).masked_fill(~seen, -math.inf), -1)
            want[i, :n, h] = w @ vv
            # A score is off by at most 2^-17 (a query in two terms) and 2^-17 (128 sums in f32) of the products' sizes, a weight by twice that, the
            # split of the weight and the exponential by 2^-16, a sum over n keys by 2^-23 for each 16 of them
            size = (qq.abs() @ kk.abs().T * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            wide = w @ vv.abs()
            slack[i, :n, h] = wide * (2.0 ** -15 * size + 2.0 ** -15 + (p + n) * 2.0 ** -27)
            if q.dtype == torch.bfloat16:  # a weight and the result are rounded to bf16
                slack[i, :n, h] += 2.0 ** -8 * wide + 2.0 ** -8 * want[i, :n, h].abs()
    return want, slack


def check(ctx, args, scale=None, **how):
    import torch
    from lemonade_burn_b200 import ops
    q, k, v, pos, parents, counts = args
    old = torch.full_like(q, 7.0)
    got = ops.attn_tree(q, k, v, *dev(pos, parents, counts), scale=scale, out=old.clone(), **how)
    ctx.check_device_error()
    want, slack = expected(q, k, v, pos, parents, counts, HD ** -0.5 if scale is None else scale)
    unused = want.isnan()
    assert torch.equal(got[unused], old[unused])
    off = (got.double() - want).abs()[~unused]
    assert bool((off <= slack[~unused]).all()), f"off by {float((off / slack[~unused]).max())} of what is allowed"
    rel = float(off.norm() / want[~unused].norm()) if off.numel() else 0.0
    assert rel < (1e-5 if q.dtype == torch.float32 else 5e-3)
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("b,t,nh,kvh,lengths", [
    (1, 1, 20, 5, [0]), (1, 1, 20, 5, [1]), (1, 1, 1, 1, [63]), (1, 1, 20, 5, [64]), (1, 1, 9, 1, [300]), (1, 2, 8, 8, [62]), (1, 5, 20, 5, [4001]), (2, 4, 16, 4, [0, 127]),
    (1, 7, 20, 5, [129]), (3, 8, 32, 8, [5, 700, 64]), (1, 16, 20, 5, [1000]), (1, 64, 20, 5, [0]), (2, 33, 20, 5, [61, 3000]), (1, 128, 8, 8, [100]), (1, 128, 20, 5, [1]),
    (1, 100, 9, 1, [2000]), (1, 3, 32, 1, [77]), (1, 37, 40, 2, [513])])
def test_attention(ctx, dtype, b, t, nh, kvh, lengths):
    import torch
    check(ctx, make(b, t, nh, kvh, lengths, getattr(torch, dtype)))


@pytest.mark.parametrize("shape", ["chain", "star", "roots"])
@pytest.mark.parametrize("t", [3, 70, 128])
def test_trees(ctx, shape, t):
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        check(ctx, make(2, t, 4, 2, [10, 100], dtype, shape))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("t,nh,kvh", [(1, 20, 5), (6, 20, 5), (26, 20, 5), (40, 8, 8)])
def test_ragged_batches(ctx, dtype, t, nh, kvh):
    """Sequences of all lengths, some without nodes, some with fewer than there are places for."""
    import torch
    lengths = [0, 1, 64, 500, 63, 128, 2500, 17, 900, 65, 3]
    counts = [t, 0, 1, t, max(1, t - 3), t, t, max(1, t // 2), 0, 1, t]
    check(ctx, make(11, t, nh, kvh, lengths, getattr(torch, dtype), counts=counts))


def test_nothing_to_do(ctx):
    import torch
    check(ctx, make(3, 4, 4, 1, [5, 0, 9], torch.float32, counts=[0, 0, 0]))


def test_many_sequences(ctx):
    import torch
    lengths = [(37 * i) % 150 for i in range(200)]
    check(ctx, make(200, 3, 2, 1, lengths, torch.float32, counts=[i % 4 for i in range(200)]))


@pytest.mark.parametrize("length", [20000, 70000])
@pytest.mark.parametrize("t", [2, 50])
def test_long_caches(ctx, length, t):
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        check(ctx, make(1, t, 4, 1, [length], dtype))


def test_offsets_past_32_bits(ctx):
    """The last sequence's rows lie 4.5 GB behind the first one's."""
    import torch
    from lemonade_burn_b200 import ops
    b, t, nh, kvh, cap = 2, 5, 16, 8, 1100000
    q, k, v, pos, parents, counts = make(b, t, nh, kvh, [3, 200], torch.float32)
    big = [torch.empty(b, kvh, cap, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, y in zip(big, (k, v)):
        x[:, :, :y.shape[2]] = y
    for short in (0, cap - 300):
        at = pos.clone()
        if short:  # the last rows of the last slab, everything in front of them as it is
            big[0][1, :, short:short + y.shape[2]], big[1][1, :, short:short + y.shape[2]] = k[1], v[1]
            big[0][1, :, :short], big[1][1, :, :short] = 0.0, 1.0
            at[1] += short
        got = ops.attn_tree(q, *big, *dev(at, parents, counts))
        ctx.check_device_error()
        if not short:
            want, slack = expected(q, k, v, pos, parents, counts)
            assert bool(((got.double() - want).abs() <= slack).all())
        else:  # `short` keys of zero scores and values of one, then the others
            for h in (0, nh - 1):
                kk, vv, qq = k[1, h // 2].double(), v[1, h // 2].double(), q[1, :, h].double()
                sc = qq @ kk[:205].T * HD ** -0.5
                for node in range(t):
                    rows = list(range(200)) + [200 + a for a in chain(parents[1], node)]
                    e = torch.exp(sc[node, rows])
                    want = (e @ vv[rows] + short) / (e.sum() + short)
                    # the same bound as `expected`, with the sum over the keys of one worker
                    assert bool(((got[1, node, h].double() - want).abs() <= 2.0 ** -12 + cap / 148 * 2.0 ** -27).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("t,nh,kvh,length", [(3, 4, 1, 10), (8, 20, 5, 200), (60, 8, 2, 130), (128, 4, 1, 40)])
def test_values_that_are_no_numbers(ctx, dtype, t, nh, kvh, length):
    """Keys and values of a branch are infinite or NaN: the other branches do not notice, the branch itself does."""
    import torch
    from lemonade_burn_b200 import ops
    dt = getattr(torch, dtype)
    q, k, v, pos, parents, counts = make(1, t, nh, kvh, [length], dt, "random")
    parents[0, t - 1] = 0
    parents[0, 1] = 0
    clean = ops.attn_tree(q, k, v, *dev(pos, parents, counts))
    sees = lambda n: torch.tensor([n in chain(parents[0], i) for i in range(t)], device="cuda")  # noqa: E731
    for where, value in (("v", math.nan), ("v", math.inf), ("v", -math.inf), ("k", math.nan), ("both", math.nan), ("k", math.inf)):
        for node in (1, t - 1):
            k2, v2 = k.clone(), v.clone()
            if where in ("k", "both"):
                k2[:, :, length + node, 5] = value
            if where in ("v", "both"):
                v2[:, :, length + node, 9] = value
            got = ops.attn_tree(q, k2, v2, *dev(pos, parents, counts))
            ctx.check_device_error()
            hit = sees(node)
            assert torch.equal(got[:, ~hit], clean[:, ~hit])
            if where == "v":
                rest = torch.arange(HD, device="cuda") != 9
                assert torch.equal(got[..., rest], clean[..., rest])
                seen = got[:, hit][..., 9]
                assert bool(seen.isnan().all() if math.isnan(value) else (seen == value).all())
            elif math.isnan(value):
                assert bool(got[:, hit].isnan().all())
    v2 = v.clone()
    v2[:, :, length + 1, 3], v2[:, :, length + t - 1, 3] = math.inf, -math.inf   # each branch its own
    got = ops.attn_tree(q, k, v2, *dev(pos, parents, counts))
    for node, value in ((1, math.inf), (t - 1, -math.inf)):
        only = sees(node) & ~sees(t - 1 if node == 1 else 1)
        assert bool((got[:, only][..., 3] == value).all())
    v2 = v.clone()
    v2[:, :, length - 1, 3] = math.nan                                             # a committed row is everybody's
    assert bool(ops.attn_tree(q, k, v2, *dev(pos, parents, counts))[..., 3].isnan().all())


def test_a_query_that_is_no_number(ctx):
    import torch
    from lemonade_burn_b200 import ops
    for t in (4, 40):
        q, k, v, pos, parents, counts = make(1, t, 4, 2, [90], torch.float32)
        clean = ops.attn_tree(q, k, v, *dev(pos, parents, counts))
        q2 = q.clone()
        q2[0, 2, 1, 7], q2[0, 3, 0, 0] = math.nan, math.inf
        got = ops.attn_tree(q2, k, v, *dev(pos, parents, counts))
        assert bool(got[0, 2, 1].isnan().all())
        same = torch.ones(t, 4, dtype=torch.bool, device="cuda")
        same[2, 1] = same[3, 0] = False
        assert torch.equal(got[0][same], clean[0][same])


def test_scores_far_apart(ctx):
    """Maxima that grow from block to block, and scores so large that only one key counts."""
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        for t in (3, 30):
            q, k, v, pos, parents, counts = make(1, t, 4, 1, [700], dtype)
            grow = torch.linspace(0.01, 6.0, k.shape[2], device="cuda")[:, None]
            k = torch.where(k.isnan(), k, (q[0, 0, 0].float() * grow).to(torch.bfloat16) + k)
            from lemonade_burn_b200 import ops
            got = ops.attn_tree(q, k, v, *dev(pos, parents, counts))
            want, slack = expected(q, k, v, pos, parents, counts)
            assert bool(((got.double() - want).abs() <= slack).all())


@pytest.mark.parametrize("scale", [1e-3, 0.3])
def test_scales(ctx, scale):
    import torch
    check(ctx, make(2, 9, 8, 2, [300, 20], torch.float32, spread=0.7), scale=scale)


@pytest.mark.parametrize("dtype,gap", [("float32", 4), ("float32", 400), ("bfloat16", 8)])
def test_strides(ctx, dtype, gap):
    import torch
    from lemonade_burn_b200 import ops
    for b, t in ((3, 5), (3, 1), (1, 6), (1, 1)):
        q, k, v, pos, parents, counts = make(b, t, 4, 2, [40] * b, getattr(torch, dtype))
        wide, room = (torch.full((b, t, 4 * HD + gap), 3.0, dtype=q.dtype, device="cuda") for _ in range(2))
        wide[..., :4 * HD] = q.view(b, t, -1)
        inside = lambda x: x[..., :4 * HD].view(b, t, 4, HD)  # noqa: E731
        ops.attn_tree(inside(wide), k, v, *dev(pos, parents, counts), out=inside(room))
        assert torch.equal(inside(room), ops.attn_tree(q, k, v, *dev(pos, parents, counts)))
        assert bool((room[..., 4 * HD:] == 3.0).all())


def test_bits_do_not_change_from_run_to_run(ctx):
    import torch
    from lemonade_burn_b200 import ops
    args = make(3, 20, 20, 5, [900, 2000, 10], torch.float32)
    first = ops.attn_tree(*args[:3], *dev(*args[3:]))
    for _ in range(20):
        assert torch.equal(ops.attn_tree(*args[:3], *dev(*args[3:])), first)


@pytest.mark.parametrize("b,t,nh,kvh,length", [(16, 4, 20, 5, 4000), (16, 8, 20, 5, 3000), (16, 16, 32, 8, 1500), (9, 128, 8, 2, 2000), (1, 6, 4, 1, 60000)])
def test_long_walks_over_and_over(ctx, b, t, nh, kvh, length):
    """Every worker has tens of blocks of several tiles: its roles run far apart, and each wait has to end."""
    import torch
    from lemonade_burn_b200 import ops
    for dtype in (torch.float32, torch.bfloat16):
        args = make(b, t, nh, kvh, [length - (7 * i) % 300 for i in range(b)], dtype)
        on = dev(*args[3:])
        first = ops.attn_tree(*args[:3], *on)
        for _ in range(60):
            got = ops.attn_tree(*args[:3], *on)
        assert torch.equal(got, first)
        ctx.check_device_error()
    check(ctx, args)


def test_bad_positions_and_parents(ctx):
    import torch
    from lemonade_burn_b200 import _lib, ops
    q, k, v, pos, parents, counts = make(3, 6, 4, 2, [30, 30, 30], torch.float32)
    clean = ops.attn_tree(q, k, v, *dev(pos, parents, counts))
    cap = k.shape[2]
    for bad in (-1, cap - 5, 2 ** 31 - 1, -2 ** 31):
        at = ints([30, bad, 30])
        out = torch.full_like(q, 5.0)
        ops.attn_tree(q, k, v, *dev(at, parents, counts), out=out)
        with pytest.raises(_lib.LbkError) as e:
            ctx.check_device_error()
        assert e.value.status == 1 and bool((out[1] == 5.0).all()) and bool((out[[0, 2]] - clean[[0, 2]]).abs().max() < 1e-5)
    for bad in (3, 5, -2, 2 ** 31 - 1, -2 ** 31):
        wrong, right = parents.clone(), parents.clone()
        wrong[1, 3], right[1, 3] = bad, -1
        out = ops.attn_tree(q, k, v, *dev(pos, wrong, counts))
        with pytest.raises(_lib.LbkError):
            ctx.check_device_error()
        assert torch.equal(out, ops.attn_tree(q, k, v, *dev(pos, right, counts)))
    for count, as_if in ((-3, 0), (9, 6)):  # a count outside the places is the nearest one inside
        out, other = torch.full_like(q, 5.0), torch.full_like(q, 5.0)
        ops.attn_tree(q, k, v, *dev(pos, parents, ints([6, count, 6])), out=out)
        ops.attn_tree(q, k, v, *dev(pos, parents, ints([6, as_if, 6])), out=other)
        assert torch.equal(out, other)
    ctx.check_device_error()


def test_refusals(ctx):
    import torch
    from lemonade_burn_b200 import _lib, ops
    q, k, v, pos, parents, counts = make(2, 4, 4, 2, [10, 20], torch.float32)
    on = dev(pos, parents, counts)
    with pytest.raises(TypeError):
        ops.attn_tree(q.half(), k, v, *on)
    for bad in (q[:1], q[:, :3], q[..., :64], q.transpose(1, 2), q[:, :, :3]):
        with pytest.raises(ValueError):
            ops.attn_tree(bad, k, v, *on)
    with pytest.raises(ValueError):
        ops.attn_tree(q, k, v, *on, out=torch.empty_like(q).to(torch.bfloat16))
    with pytest.raises(ValueError):
        ops.attn_tree(q, k.transpose(1, 2).contiguous().transpose(1, 2), v, *on)
    with pytest.raises(ValueError):
        ops.attn_tree(q, k, v, pos, *on[1:])
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    scratch, out = torch.empty(lib.lbk_attn_tree_scratch(ctx.handle, 4, 4, 2), device="cuda"), torch.empty_like(q)
    good = dict(compute=1, q=q.data_ptr(), pitch=512, t=4, nh=4, kvh=2, hd=128, scale=1.0, scratch=scratch.data_ptr(), out=out.data_ptr(), out_pitch=512, b=2)

    def call(**change):
        a = {**good, **change}
        return lib.lbk_attn_tree(ctx.handle, a["compute"], a["q"], a["pitch"], k.data_ptr(), v.data_ptr(), *[x.data_ptr() for x in on], a["b"], a["t"], a["nh"], a["kvh"], a["hd"],
                                 k.shape[2], a["scale"], a["scratch"], a["out"], a["out_pitch"], st)
    assert call() == 0 and call(b=0) == 0
    for change, status in ((dict(compute=2), 1), (dict(q=None), 1), (dict(scratch=None), 1), (dict(t=129), 4), (dict(b=257), 4), (dict(hd=64), 2), (dict(kvh=3), 2), (dict(kvh=0), 2),
                           (dict(scale=0.0), 1), (dict(scale=math.nan), 1), (dict(pitch=508), 2), (dict(pitch=514), 2), (dict(out_pitch=511), 2), (dict(q=q.data_ptr() + 4), 2),
                           (dict(out=out.data_ptr() + 8), 2), (dict(compute=0, pitch=516), 2)):
        assert call(**change) == status, change
    ctx.check_device_error()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("b,t,nh,kvh,lengths", [(256, 1, 2, 1, [i % 3 for i in range(256)]), (1, 2, 4096, 1, [70]), (1, 1, 4096, 4096, [3]), (2, 128, 32, 1, [5, 130])])
def test_the_largest_batches_and_heads(ctx, dtype, b, t, nh, kvh, lengths):
    import torch
    check(ctx, make(b, t, nh, kvh, lengths, getattr(torch, dtype)))


@pytest.mark.parametrize("t,nh", [(1, 4), (5, 16), (40, 8)])
def test_a_cache_without_room_to_spare(ctx, t, nh):
    """The last node's row is the cache's last one, and the sequence the buffer's last."""
    import torch
    for pos in (0, 1, 60, 130):
        q, k, v, lengths, parents, counts = make(2, t, nh, 2, [pos, pos], torch.float32)
        check(ctx, (q, k[:, :, :pos + t].contiguous(), v[:, :, :pos + t].contiguous(), lengths, parents, counts))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("b,t,nh,kvh,length", [(1, 1, 20, 5, 900), (2, 6, 20, 5, 5000), (1, 60, 8, 2, 9000), (3, 128, 8, 2, 100)])
def test_results_in_the_place_of_the_queries(ctx, dtype, b, t, nh, kvh, length):
    import torch
    from lemonade_burn_b200 import ops
    q, k, v, pos, parents, counts = make(b, t, nh, kvh, [length] * b, getattr(torch, dtype))
    on = dev(pos, parents, counts)
    want = ops.attn_tree(q, k, v, *on, out=q.clone())  # rows of places not in use stay
    assert ops.attn_tree(q, k, v, *on, out=q) is q and torch.equal(q, want)
    ctx.check_device_error()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_that_are_no_numbers_where_the_walk_goes_round(ctx, dtype):
    """Two tiles a head and many blocks a worker: the nodes' block comes up in the middle of a walk."""
    test_values_that_are_no_numbers(ctx, dtype, 60, 8, 2, 40000)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_walks_that_go_round(ctx, dtype):
    import torch
    for b, t, nh, kvh, lengths in ((1, 70, 8, 2, [30011]), (3, 100, 4, 1, [9000, 0, 20500]), (40, 65, 4, 2, [700 + 37 * i for i in range(40)])):
        check(ctx, make(b, t, nh, kvh, lengths, getattr(torch, dtype), counts=[t - i % 3 for i in range(b)]))
