"""Drafted tokens and scores where numbers lie at the ends of their ranges: a NaN at the first token, paths that are none, tokens outside the
vocabulary, scores of texts of all lengths."""
import math

import pytest

from test_gpu_draft import _check_logprobs, dev, ints, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,shift", [(12, 4, 0), (12, 20, 0), (12, 32, 1), (12, 33, 3), (12, 700, 1), (600, 700, 1), (12, 9001, 0), (600, 2500, 1), (12, 130001, 3), (200, 40000, 0)])
def test_a_nan_at_the_first_token(ctx, dtype, rows, vocab, shift):
    """It is the first alternative: alone, among others, in rows of nothing else. In rows of a warp, of a block and of a cluster; in a vector of loads and in front of the first."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(rows, vocab + shift, generator=g, device="cuda")[:, shift:]
    x[::6, 0] = math.nan
    x[1::6] = math.nan
    x[2::6, :3] = math.nan
    x[3::6, 0], x[3::6, 1] = math.nan, math.inf
    x[4::6, 1:], x[4::6, 0] = -math.inf, math.nan
    x[5::6, vocab - 1] = math.nan
    wide = torch.empty(rows, vocab + shift, dtype=getattr(torch, dtype), device="cuda")
    wide[:, shift:] = x
    x = wide[:, shift:]
    tokens = torch.tensor([[0, vocab - 1]], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous()
    for top in {1, min(vocab, 5), min(vocab, 32)}:
        _check_logprobs(x, tokens, top)


def test_a_path_that_is_none_commits_nothing(ctx):
    """A sampler's path that does not ascend, leaves the tree or the cache: neither rows nor position of that sequence move; the others' do."""
    import torch
    from lemonade_burn_b200 import _lib
    from test_gpu_draft_models import small
    net = small(ctx, layers=2, max_pos=40)
    for path, count, at in (([1, 0, -1, -1], 2, 9), ([0, 0, 1, -1], 3, 9), ([0, 4, -1, -1], 2, 9), ([-1, 1, -1, -1], 2, 9), ([0, 1, 3, -1], 3, 37), ([0, 1, 3, -1], 3, -1), ([0, 2, 3, -1], 4, 9)):
        cache = net.new_cache(3, 40, own_positions=True)
        cache.k.normal_()
        cache.v.normal_()
        cache.pos.copy_(ints([5, at, 7]))
        old = cache.k.clone(), cache.v.clone()
        net.accept_tree(cache, *dev(ints([[0, 3, -1, -1], path, [2, -1, -1, -1]]), ints([2, count, 1])))
        with pytest.raises(_lib.LbkError) as e:
            ctx.check_device_error()
        assert e.value.status == 1
        assert cache.pos.tolist() == [7, at, 8]
        for now, was in zip((cache.k, cache.v), old):
            assert torch.equal(now[:, 1], was[:, 1])
            assert torch.equal(now[:, 0, :, 6], was[:, 0, :, 8]) and torch.equal(now[:, 2, :, 7], was[:, 2, :, 9])


def test_counts_outside_the_tree_are_the_nearest_inside(ctx):
    """What keeps the rows and what moves the position take a count alike."""
    from test_gpu_draft_models import small
    net = small(ctx, layers=1, max_pos=40)
    cache = net.new_cache(4, 40, own_positions=True)
    cache.pos.fill_(5)
    net.accept_tree(cache, *dev(ints([[0, 1, 2]] * 4), ints([100, -3, 2 ** 31 - 1, 3])))
    ctx.check_device_error()
    assert cache.lens() == [8, 5, 8, 8] and cache.host_len >= 3


@pytest.mark.parametrize("b,t", [(1, 1), (5, 128), (9, 70), (300, 33)])
def test_keep_and_advance_in_one_call(ctx, b, t):
    import torch
    from lemonade_burn_b200 import ops
    g = torch.Generator().manual_seed(b)
    cap, count = t + 4, [(i * 7) % (t + 1) for i in range(b)]
    path = torch.full((b, t), -1, dtype=torch.int32)
    for i, n in enumerate(count):
        path[i, :n] = torch.randperm(t, generator=g)[:n].sort().values.int()
    k = torch.randn(2, b, 1, cap, 8, device="cuda").to(torch.bfloat16)
    v, pos, moved = k + 1, *dev(ints([i % 5 for i in range(b)]), ints([i % 5 for i in range(b)]))
    k2, v2 = k.clone(), v.clone()
    ops.kv_keep_path(k, v, pos, *dev(path, ints(count)))
    ops.kv_keep_path(k2, v2, moved, *dev(path, ints(count)), advance=True)
    assert torch.equal(k, k2) and torch.equal(v, v2) and pos.tolist() == [i % 5 for i in range(b)] and moved.tolist() == [i % 5 + n for i, n in enumerate(count)]
    ctx.check_device_error()


@pytest.mark.parametrize("heads,vocab", [(4, 700), (2, 300)])
def test_places_that_are_not_in_use_hold_anything(ctx, heads, vocab):
    """A batch of trees of different sizes is padded with whatever was there: with -1, as paths and `after` of a sequence without nodes are, or with any number."""
    import torch
    from test_gpu_draft_models import near, small
    net = small(ctx, heads=heads, layers=2, vocab=vocab)
    b, t = 4, 6
    g = torch.Generator().manual_seed(1)
    counts = ints([3, 0, 6, 1])
    tokens, parents = torch.randint(0, vocab, (b, t), generator=g, dtype=torch.int32), trees(b, t, 2)
    unused = torch.arange(t) >= counts[:, None]
    results = []
    for fill in (0, -1, 2 ** 31 - 1, -2 ** 31, vocab):
        padded = torch.where(unused, torch.tensor(fill, dtype=torch.int32), tokens)
        at = torch.where(unused, torch.tensor(fill, dtype=torch.int32), parents)
        cache = net.new_cache(b, 64, own_positions=True)
        logits = net.forward_tree(*dev(padded, at), cache, counts.cuda())
        assert bool(logits.isfinite().all())
        path, count, after = net.decode_tree(*dev(padded, at), cache, counts.cuda())
        results.append((logits[~unused], path, count, after, cache.k, cache.v))
        ctx.check_device_error()
    for r in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, results[0]))
    alone = net.forward_tree(tokens[2:3].cuda(), parents[2:3].cuda(), net.new_cache(1, 64))
    assert near(results[0][0][-7:-1], alone[0])


def test_tokens_outside_the_vocabulary_are_reported(ctx):
    import torch
    from lemonade_burn_b200 import _lib
    from test_gpu_draft_models import near, small
    net = small(ctx, layers=1)
    for bad in (-1, 700, 2 ** 31 - 1, -2 ** 31):
        tokens, parents = ints([[5, 6, 7], [5, bad, 7]]), trees(2, 3, 0, "star")
        cache = net.new_cache(2, 32, own_positions=True)
        logits = net.forward_tree(*dev(tokens, parents), cache)
        with pytest.raises(_lib.LbkError) as e:
            ctx.check_device_error()
        assert e.value.status == 1 and "vocabulary" in str(e.value)
        assert near(logits[0], net.forward_tree(tokens[:1].cuda(), parents[:1].cuda(), net.new_cache(1, 32))[0])
    for counts in (torch.zeros(2, dtype=torch.int64), ints([1]), ints([[1, 1]])):
        with pytest.raises(ValueError, match="counts"):
            net.forward_tree(*dev(ints([[1], [2]]), ints([[-1], [-1]])), net.new_cache(2, 32, own_positions=True), counts.cuda())
    ctx.check_device_error()


@pytest.mark.parametrize("hidden,shift", [(64, 0), (512, 0), (2560, 0), (514, 0), (33, 0), (512, 1)])
@pytest.mark.parametrize("b,t", [(1, 1), (3, 7), (9, 128)])
def test_rows_of_nodes(ctx, hidden, shift, b, t):
    """The rows of the call for one token a sequence, bit by bit; the form by four and the form by one."""
    import torch
    from lemonade_burn_b200 import _lib
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    g = torch.Generator(device="cuda").manual_seed(hidden)
    table = torch.randn(301 * hidden + shift, generator=g, device="cuda").to(torch.bfloat16)[shift:].view(301, hidden)
    tokens = torch.randint(0, 301, (b, t), generator=g, device="cuda", dtype=torch.int32)
    counts = [(3 * i + 1) % (t + 1) for i in range(b)]
    out = torch.empty(b, t, hidden, device="cuda")
    for c in (None, ints(counts).cuda()):
        _lib.check(lib.lbk_embed_tree_bf16(ctx.handle, table.data_ptr(), 301, tokens.data_ptr(), None if c is None else c.data_ptr(), b, t, hidden, out.data_ptr(), st))
        want = table[tokens.long()].float()
        if c is not None:
            want[torch.arange(t, device="cuda") >= c[:, None]] = table[0].float()
        assert torch.equal(out, want)
    assert lib.lbk_embed_tree_bf16(ctx.handle, table.data_ptr(), 0, tokens.data_ptr(), None, b, t, hidden, out.data_ptr(), st) == 2
    assert lib.lbk_embed_tree_bf16(ctx.handle, table.data_ptr(), 301, tokens.data_ptr(), None, b, 129, hidden, out.data_ptr(), st) == 4
    assert lib.lbk_embed_tree_bf16(ctx.handle, None, 301, tokens.data_ptr(), None, b, t, hidden, out.data_ptr(), st) == 1
    ctx.check_device_error()


def test_scores_of_texts_of_all_lengths_take_no_more_memory_than_the_longest(ctx, tmp_path):
    """A cache that is reset and scored with longer and longer texts."""
    import numpy as np
    import torch
    from lemonade_burn_b200 import model
    longest = 1200
    cfg = model.Config(256, 384, 2, 1, 1, 300, 1e-5, 500000.0, 2048)
    model.save_checkpoint(tmp_path, cfg, model.random_checkpoint(cfg, 8))
    net = model.NativeBitNet(tmp_path, ctx)
    toks = np.random.default_rng(0).integers(0, 300, longest).astype(np.uint32)
    net.score(toks, net.new_cache(1, longest), top=20)  # what the library itself keeps

    def room(lengths):
        cache = net.new_cache(1, longest)
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        for n in lengths:
            net.reset_cache(cache)
            scores = net.score(toks[:n], cache, top=20)
        return before - torch.cuda.mem_get_info()[0], scores
    alone, want = room([longest])
    grown, got = room(range(1, longest + 1))
    # 1, 2, .., 1200 rows of 43 words are 124 MB; the allocator's pages are 2 MB
    assert grown <= alone + (16 << 20)
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(got, want))
    net.close()


@pytest.mark.parametrize("layers,one_launch", [(1, True), (2, False)])
def test_a_step_with_a_token_outside_the_vocabulary(ctx, layers, one_launch):
    """decode_tree gives -1 for a sequence without nodes; a step that is handed it reads no row in front of the table, and the other sequences do not notice."""
    import torch
    from lemonade_burn_b200 import _lib
    from test_gpu_draft_models import small
    net = small(ctx, layers=layers)
    how = {} if one_launch else {"splits": 2}
    cache = net.new_cache(2, 32, own_positions=True)
    _, count, after = net.decode_tree(*dev(ints([[5, 6], [7, 8]]), ints([[-1, 0], [-1, 0]])), cache, ints([2, 0]).cuda())
    assert int(after[1]) == -1 and int(count[1]) == 0
    ctx.check_device_error()
    got = net.forward(after, cache, **how)
    with pytest.raises(_lib.LbkError) as e:
        ctx.check_device_error()
    assert "vocabulary" in str(e.value) and bool(got.isfinite().all())
    for token in (0, 700, 2 ** 31 - 1, -2 ** 31):
        other = net.new_cache(2, 32, own_positions=True)
        net.decode_tree(*dev(ints([[5, 6], [7, 8]]), ints([[-1, 0], [-1, 0]])), other, ints([2, 0]).cuda())
        assert torch.equal(net.forward(torch.stack([after[0], torch.tensor(token, dtype=torch.int32, device="cuda")]), other, **how), got)
        if token:
            with pytest.raises(_lib.LbkError):
                ctx.check_device_error()
    ctx.check_device_error()
