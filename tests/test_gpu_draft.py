"""Drafted tokens: append by depth, the greedy walk, moving accepted rows together, log probabilities; each against plain loops in
64 bits, at the sizes, masks and values where it can go wrong."""
import math

import pytest

pytestmark = pytest.mark.gpu


def trees(b, t, seed, shape="random"):
    """Parents [b, t] int32 on the CPU: a chain, a star, several roots, or nodes hung on any node in front of them."""
    import torch
    g = torch.Generator().manual_seed(seed)
    at = torch.arange(t)
    if shape == "chain":
        p = (at - 1).expand(b, t)
    elif shape == "star":
        p = torch.zeros(b, t, dtype=torch.long)
    elif shape == "roots":
        p = torch.where(torch.rand(b, t, generator=g) < 0.3, -1, (torch.rand(b, t, generator=g) * at).long())
    else:
        p = (torch.rand(b, t, generator=g) * at).long()
    p = p.clone()
    p[:, 0] = -1
    return p.int()


def chain(parents, i):
    found = []
    while i >= 0:
        found.append(i)
        i = int(parents[i])
    return found


def dev(*ts):
    return [None if t is None else t.cuda() for t in ts]


def ints(v):
    import torch
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("hd,nh,kvh", [(128, 20, 5), (128, 1, 1), (64, 3, 3), (8, 4, 2), (12, 5, 1), (2, 1, 1), (256, 2, 1)])
@pytest.mark.parametrize("b,t,shape", [(1, 1, "chain"), (3, 5, "chain"), (2, 128, "chain"), (4, 33, "random"), (2, 17, "roots")])
def test_append(ctx, hd, nh, kvh, b, t, shape):
    import torch
    from lemonade_burn_b200 import ops
    cap = t + 9
    parents = trees(b, t, 3 * t + hd, shape)
    counts = None if b == 1 else ints([0 if i == 1 else max(1, t - 2 * i) for i in range(b)])
    pos = ints([(4 * i) % 9 for i in range(b)])
    g = torch.Generator(device="cuda").manual_seed(hd + t)
    q, k, v, cos, sin = (torch.randn(s, generator=g, device="cuda") for s in ((b, t, nh * hd), (b, t, kvh * hd), (b, t, kvh * hd), (cap, hd), (cap, hd)))
    kc, vc = (torch.randn(b, kvh, cap, hd, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    want_q, size_q, want_k, size_k, want_v = q.double().view(b, t, nh, hd).clone(), torch.zeros(b, t, nh, hd, device="cuda").double(), kc.double(), torch.zeros_like(kc).double(), vc.clone()
    half = hd // 2
    for i in range(b):
        for n in range(t if counts is None else int(counts[i])):
            place, row = int(pos[i]) + len(chain(parents[i], n)) - 1, int(pos[i]) + n
            c, s = cos[place].double(), sin[place].double()
            turn = lambda x: (x * c, torch.cat([-x[..., half:], x[..., :half]], -1) * s)  # noqa: E731
            a, o = turn(q[i, n].double().view(nh, hd))
            want_q[i, n], size_q[i, n] = a + o, a.abs() + o.abs()
            a, o = turn(k[i, n].double().view(kvh, hd))
            want_k[i, :, row], size_k[i, :, row] = a + o, a.abs() + o.abs()
            want_v[i, :, row] = v[i, n].view(kvh, hd).to(torch.bfloat16)
    ops.rope_kv_append_tree(q, k, v, cos, sin, *dev(pos, parents), kc, vc, counts=dev(counts)[0])
    ctx.check_device_error()
    # a product and the sum, each rounded once: 2^-24 of each; keys are rounded to bf16 too. Untouched places are the same bits.
    assert bool(((q.view(b, t, nh, hd).double() - want_q).abs() <= 2.0 ** -23 * size_q).all())
    assert bool(((kc.double() - want_k).abs() <= 2.0 ** -22 * size_k + 2.0 ** -8 * want_k.abs() * (size_k > 0)).all())
    assert torch.equal(vc, want_v)


def test_append_of_buffers_off_16_bytes(ctx):
    """The form value by value gives the bits of the form by four."""
    import torch
    from lemonade_burn_b200 import ops
    b, t, nh, kvh, hd, cap = 2, 9, 3, 1, 128, 20
    g = torch.Generator(device="cuda").manual_seed(5)
    data = [torch.randn(s, generator=g, device="cuda") for s in ((b, t, nh * hd), (b, t, kvh * hd), (b, t, kvh * hd), (cap, hd), (cap, hd))]
    pos, parents = dev(ints([1, 7]), trees(b, t, 1))
    got = []
    for shift in (0, 1):
        place = lambda x: torch.cat([x.new_zeros(shift), x.reshape(-1)])[shift:].view(x.shape)  # noqa: E731
        q, k, v, cos, sin = (place(x) for x in data)
        kc, vc = (place(torch.zeros(b, kvh, cap, hd, device="cuda", dtype=torch.bfloat16)) for _ in range(2))
        ops.rope_kv_append_tree(q, k, v, cos, sin, pos, parents, kc, vc)
        got.append((q, kc, vc))
    assert all(torch.equal(x, y) for x, y in zip(*got))


def walk(tokens, parents, best, count):
    if not count:
        return [], -1
    path = [0]
    while True:
        fits = [n for n in range(count) if parents[n] == path[-1] and tokens[n] == best[path[-1]]]
        if not fits:
            return path, int(best[path[-1]])
        path.append(fits[0])


@pytest.mark.parametrize("t", [1, 2, 31, 33, 64, 100, 128])
@pytest.mark.parametrize("shape", ["chain", "star", "random", "roots"])
def test_accept(ctx, t, shape):
    import torch
    from lemonade_burn_b200 import ops
    b = 5
    parents = trees(b, t, t, shape)
    g = torch.Generator().manual_seed(t)
    tokens, best = (torch.randint(0, 2, (b, t), generator=g, dtype=torch.int32) for _ in range(2))  # many twins
    best[4] = tokens[4] = 7                                                                          # the longest path there is
    for counts in (None, ints([t, 0, max(1, t // 2), 1, t])):
        path, count, after = ops.tree_accept(*dev(tokens, parents, best, counts))
        for i in range(b):
            want, last = walk(tokens[i], parents[i], best[i], t if counts is None else int(counts[i]))
            assert path[i].tolist() == want + [-1] * (t - len(want)) and int(count[i]) == len(want) and int(after[i]) == last
    ctx.check_device_error()


@pytest.mark.parametrize("layers,b,kvh,hd", [(1, 1, 1, 128), (3, 4, 5, 128), (2, 3, 2, 8), (2, 2, 1, 264)])
@pytest.mark.parametrize("t", [1, 7, 128])
def test_keep_path(ctx, layers, b, kvh, hd, t):
    import torch
    from lemonade_burn_b200 import ops
    cap = t + 11
    g = torch.Generator(device="cuda").manual_seed(t)
    k, v = (torch.randn(layers, b, kvh, cap, hd, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    cg = torch.Generator().manual_seed(t + b)
    pos = ints([(7 * i) % 12 for i in range(b)])
    path, count = torch.full((b, t), -1, dtype=torch.int32), []
    for i in range(b):
        n = [t, 0, 1, max(1, t // 2)][(i + b) % 4]                    # every node (nothing moves), none, the last one, half of them
        count.append(n)
        path[i, :n] = torch.randperm(t, generator=cg)[:n].sort().values.int() if n != 1 else t - 1
    want = [k.clone(), v.clone()]
    for i in range(b):
        p = int(pos[i])
        for w, c in zip(want, (k, v)):
            w[:, i, :, p:p + count[i]] = c[:, i][:, :, p + path[i, :count[i]].long()]
    at, counted = dev(pos, ints(count))
    ops.kv_keep_path(k, v, at, path.cuda(), counted)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    ops.advance_pos_by(at, counted)
    assert at.tolist() == [int(p) + n for p, n in zip(pos, count)]
    ctx.check_device_error()


def test_keep_path_of_layers_that_lie_apart(ctx):
    import torch
    from lemonade_burn_b200 import _lib
    layers, b, kvh, cap, hd, gap = 3, 2, 2, 9, 16, 40
    layer = b * kvh * cap * hd
    k, v = (torch.randn(layers, layer + gap, device="cuda").to(torch.bfloat16) for _ in range(2))
    want = [k.clone(), v.clone()]
    for w, c in zip(want, (k, v)):
        for i, p in enumerate((2, 3)):
            w[:, :layer].view(layers, b, kvh, cap, hd)[:, i, :, p:p + 2] = c[:, :layer].view(layers, b, kvh, cap, hd)[:, i][:, :, [p + 1, p + 3]]
    pos, path, count = dev(ints([2, 3]), ints([[1, 3, -1, -1]] * 2), ints([2, 2]))
    _lib.check(_lib.load().lbk_kv_keep_path(ctx.handle, k.data_ptr(), v.data_ptr(), layers, layer + gap, b, kvh, hd, cap, pos.data_ptr(), path.data_ptr(), count.data_ptr(), 4,
                                            torch.cuda.current_stream().cuda_stream))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_trees_and_positions_that_are_none_are_refused(ctx):
    """Bad numbers in device memory: the sequence keeps its buffers, the others are served, and the host hears of it."""
    import torch
    from lemonade_burn_b200 import _lib, ops
    b, t, nh, kvh, hd, cap = 3, 4, 2, 1, 128, 16
    for pos, parents in (([3, 13, 3], [[-1, 0, 1, 2]] * 3), ([3, -1, 3], [[-1, 0, 1, 2]] * 3), ([3, 3, 3], [[-1, 0, 1, 2], [-1, 0, 2, 1], [-1, 0, 0, 0]]),
                         ([3, 3, 3], [[-1, 0, 1, 2], [-2, 0, 0, 1], [-1, 0, 0, 0]]), ([3, 3, 3], [[-1, 0, 1, 2], [-1, 0, 0, 2 ** 31 - 1], [-1, 0, 0, 0]])):
        q, k, v, cos, sin = (torch.randn(s, device="cuda") for s in ((b, t, nh * hd), (b, t, kvh * hd), (b, t, kvh * hd), (cap, hd), (cap, hd)))
        kc, vc = (torch.zeros(b, kvh, cap, hd, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        old = q.clone()
        ops.rope_kv_append_tree(q, k, v, cos, sin, *dev(ints(pos), ints(parents)), kc, vc)
        with pytest.raises(_lib.LbkError) as e:
            ctx.check_device_error()
        assert e.value.status == 1
        assert torch.equal(q[1], old[1]) and not kc[1].any() and not vc[1].any()
        assert kc[0, :, 3:7].any() and kc[2, :, 3:7].any() and not torch.equal(q[2], old[2])
    path, count, after = ops.tree_accept(*dev(ints([[1, 1]] * 2), ints([[-1, 0], [-1, 1]]), ints([[1, 5]] * 2)))
    assert path.tolist() == [[0, 1], [-1, -1]] and count.tolist() == [2, 0] and after.tolist() == [5, -1]
    with pytest.raises(_lib.LbkError):
        ctx.check_device_error()
    for path in ([0, 0, -1, -1], [2, 1, -1, -1], [0, 4, -1, -1], [-1, 2, -1, -1]):  # not ascending, outside the tree
        k = torch.randn(1, 1, 1, cap, hd, device="cuda").to(torch.bfloat16)
        old = k.clone()
        ops.kv_keep_path(k, k.clone(), *dev(ints([5]), ints([path]), ints([2])))
        assert torch.equal(k, old)
        with pytest.raises(_lib.LbkError):
            ctx.check_device_error()
    ctx.check_device_error()


def _check_logprobs(x, tokens, top, scale=1.0):
    import torch
    from lemonade_burn_b200 import ops
    got = ops.token_logprobs(x, tokens, top, scale)
    d = x.double() * scale
    lp = torch.log_softmax(d, -1)
    n = x.shape[1]
    order = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids.long(), order)
    t = tokens.long().clamp(0, n - 1)
    want = torch.where((tokens >= 0) & (tokens < n), torch.gather(lp, 1, t), math.nan)
    # exp's argument is off by 2^-23 of itself and exp by 2^-21, a thread adds at most n / 256 values, and the result is rounded: with H <= log n
    # the average argument is below log n + 1
    slack = 2.0 ** -21 * (math.log(n) + 4) + (n / 256 + 32) * 2.0 ** -24
    for a, w in ((got.logprobs, want), (got.top_logprobs, torch.gather(lp, 1, order))):
        a = a.double()
        assert torch.equal(a.isnan(), w.isnan()) and torch.equal(a.isinf(), w.isinf())
        ok = w.isfinite()
        assert bool(((a - w).abs()[ok] <= slack + 2.0 ** -22 * w.abs()[ok]).all())
    entropy = torch.where(lp.isnan().any(-1), math.nan, torch.special.entr(lp.exp()).sum(-1))
    a = got.entropy.double()
    assert torch.equal(a.isnan(), entropy.isnan())
    ok = ~entropy.isnan()
    assert bool(((a - entropy).abs()[ok] <= slack * (math.log(n) + 2)).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,pad,top", [(1, 1, 0, 1), (3, 7, 0, 7), (2, 33, 5, 32), (300, 257, 0, 3), (2, 1000, 1, 0), (1, 8193, 0, 32), (5, 50021, 3, 20), (1, 128256, 0, 5),
                                                (20, 128256, 0, 20), (700, 2048, 8, 1)])
def test_logprobs(ctx, dtype, rows, vocab, pad, top):
    import torch
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (3 * torch.randn(rows, vocab + pad, generator=g, device="cuda")).to(getattr(torch, dtype))[:, :vocab]
    tokens = torch.randint(0, vocab, (rows, 3), generator=g, device="cuda", dtype=torch.int32)
    tokens[0, 1], tokens[rows - 1, 2] = -1, vocab
    for scale in (1.0, 0.6):
        _check_logprobs(x, tokens, top, scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [40, 5000, 130001])
def test_logprobs_of_unusual_rows(ctx, dtype, vocab):
    """Ties, rows in order, masks of -inf and of the type's lowest value, rows with a NaN or an infinity, rows with nothing."""
    _unusual_rows(dtype, vocab, 1)


@pytest.mark.parametrize("dtype,vocab", [("float32", 700), ("float32", 5003), ("bfloat16", 1100), ("bfloat16", 10001)])
def test_logprobs_of_many_unusual_rows(ctx, dtype, vocab):
    """The same where there are more rows than the SMs hold blocks: rows of a warp each."""
    _unusual_rows(dtype, vocab, 30)


def _unusual_rows(dtype, vocab, times):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(16, vocab, generator=g, device="cuda")
    x[0] = 1.5
    x[1] = torch.arange(vocab, device="cuda") * (8.0 / vocab)
    x[2] = torch.arange(vocab, 0, -1, device="cuda") * (8.0 / vocab)
    x[3] = -math.inf
    x[3, 7], x[3, 30], x[3, 2] = 1.0, 1.0, 3.0
    x[4] = torch.finfo(dt).min
    x[4, 5] = 0.5
    x[5] = torch.finfo(dt).min
    x[6] = -math.inf
    x[7, vocab // 2] = math.nan
    x[8, [3, vocab - 1]] = math.inf
    x[9] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    x[10] = (4 * x[10]).round()
    x[11, :] = 1e4
    x[11, vocab - 1] = 1.2e4
    x[12, [1, 9]] = math.nan
    x[12, 4] = math.inf
    x[13] = -math.inf
    x[13, vocab - 1] = -50.0
    x[14] = torch.randn(vocab, generator=g, device="cuda") * 1e-30
    x[15, ::2] = -math.inf
    x = x.to(dt).repeat(times, 1)
    tokens = torch.tensor([[0, vocab - 1, 7]], dtype=torch.int32, device="cuda").expand(16 * times, 3).contiguous()
    for top in (1, 20, 32):
        _check_logprobs(x, tokens, top)


def test_logprobs_without_tokens_or_alternatives(ctx):
    import torch
    from lemonade_burn_b200 import _lib, ops
    x = torch.randn(4, 100, device="cuda")
    got = ops.token_logprobs(x)
    assert got.logprobs.shape == (4, 0) and got.top_ids.shape == (4, 0) and got.entropy.shape == (4,)
    assert ops.token_logprobs(x, torch.zeros(4, dtype=torch.int32, device="cuda")).logprobs.shape == (4, 1)
    assert ops.token_logprobs(x[:0], top=3).top_ids.shape == (0, 3)
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    out = torch.empty(64, device="cuda")
    call = lambda dtype=0, pitch=100, vocab=100, scale=1.0, top=0, ids=None: lib.lbk_token_logprobs(  # noqa: E731
        ctx.handle, dtype, x.data_ptr(), pitch, 4, vocab, None, 0, scale, top, None, out.data_ptr(), ids, ids, st)
    assert call() == 0
    assert call(dtype=2) == 1 and call(pitch=99) == 2 and call(vocab=0) == 2 and call(scale=0.0) == 1 and call(scale=math.nan) == 1 and call(scale=math.inf) == 1
    assert call(top=3) == 1 and call(top=33, ids=out.data_ptr()) == 4 and call(pitch=200, vocab=101, top=102, ids=out.data_ptr()) == 2


@pytest.mark.parametrize("vocab", [50, 9000])
@pytest.mark.parametrize("scale", [1e-20, 1e-3, 7.0, 1e20])
def test_logprobs_at_any_scale(ctx, vocab, scale):
    """What the scale is for: temperatures. At the ends every value has the same weight, or one value all of it."""
    import torch
    from lemonade_burn_b200 import ops
    x = torch.randn(3, vocab, generator=torch.Generator().manual_seed(1)).cuda()
    x[1, 3], x[1, 7] = 3e38, -3e38
    tokens = torch.tensor([[0, 3], [7, 3], [1, 3]], dtype=torch.int32).cuda()
    got = ops.token_logprobs(x, tokens, top=2, scale=scale)
    factor = torch.tensor(scale, dtype=torch.float32).double().item()  # as the call has it
    want = torch.log_softmax(x.double() * factor, -1)
    entropy = -torch.where(want.exp() > 0, want.exp() * want, torch.zeros_like(want)).sum(-1)
    at = want.gather(1, tokens.long())
    # In steps of 2^-23. A log probability is (x - m) scale - log s: the product is off by 2 of itself; s, a thread's sum of 18 exponentials at most and eight
    # joins, by 13 + 2 for the exponentials; its logarithm, at most 10, by 10, and by the exponents' own error, |f| e^f < 1. Entropy is log s - scale t / s: t as s,
    # times 10, and twice sum p f^2 < 60 for the exponents.
    finite = at.abs() < 3e38  # f32 ends there
    assert bool(((got.logprobs.double() - at).abs() <= 2.0 ** -23 * (4 * at.abs() + 40))[finite].all()) and bool((got.logprobs[~finite] < -3e38).all())
    assert bool(((got.entropy.double() - entropy).abs() <= 2.0 ** -23 * 400).all())
    assert got.top_ids[1, 0] == 3 and torch.equal(got.top_ids.cpu().long(), x.cpu().topk(2).indices)


def test_logprobs_of_scales_that_are_none(ctx):
    import torch
    from lemonade_burn_b200 import _lib, ops
    for scale in (0.0, -1.0, 9e-21, 2e20, 3e38, 1e300, math.inf, math.nan):
        with pytest.raises(_lib.LbkError):
            ops.token_logprobs(torch.zeros(2, 9, device="cuda"), scale=scale)
