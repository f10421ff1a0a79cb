"""Drafted tokens and scores through the models: a tree's pass against the tokens one by one, accepted paths, sequences of different
lengths, recorded steps, calls on two streams; scores of all families against their logits."""
import math

import numpy as np
import pytest

from test_gpu_draft import chain, dev, ints, trees, walk

pytestmark = pytest.mark.gpu
TOL = 2e-3  # of the largest logit: the decoder's bar between its routes (int8 rounding flips)


def small(ctx, seed=3, layers=3, vocab=700, heads=4, kv=1, max_pos=96, ff=768):
    from lemonade_burn_b200 import model
    cfg = model.Config(heads * 128, ff, heads, kv, layers, vocab, 1e-5, 500000.0, max_pos)
    return model.BitNet(cfg, model.random_checkpoint(cfg, seed), ctx)


def near(got, want):
    return float((got.double() - want.double()).abs().max()) <= TOL * float(want.abs().max())


@pytest.mark.parametrize("heads,kv,ff,b,t", [(4, 1, 768, 1, 1), (4, 1, 768, 1, 5), (4, 2, 768, 3, 7), (5, 5, 1000, 2, 20), (4, 1, 8200, 2, 3), (20, 5, 768, 1, 40)])
def test_a_tree_is_its_paths_one_by_one(ctx, heads, kv, ff, b, t):
    import torch
    net = small(ctx, heads=heads, kv=kv, ff=ff)
    g = torch.Generator().manual_seed(t)
    V = net.cfg.vocab_size
    prompt = torch.randint(0, V, (6, b), generator=g, dtype=torch.int32)
    cache = net.new_cache(b, 64, own_positions=True)
    for toks in prompt:
        net.forward(toks.cuda(), cache)
    tokens, parents = torch.randint(0, V, (b, t), generator=g, dtype=torch.int32), trees(b, t, t, "roots")
    logits = net.forward_tree(*dev(tokens, parents), cache)
    assert cache.lens() == [6] * b and logits.shape == (b, t, V)
    for s in range(b):
        for node in {0, t - 1, t // 2}:
            alone = net.new_cache(1, 64)
            for toks in prompt:
                net.forward(toks[s:s + 1].cuda(), alone)
            for n in reversed(chain(parents[s], node)):
                want = net.forward(tokens[s, n:n + 1].cuda(), alone)[0]
            assert near(logits[s, node], want)
    ctx.check_device_error()


def test_steps_with_drafts_leave_the_cache_of_steps_without(ctx):
    """Trees of a ragged batch, some guesses right and some wrong: what is accepted follows from the trees' own logits, and cache, positions and
    the next tokens' logits are those of the accepted tokens one by one."""
    import torch
    net, b, t, cap = small(ctx, seed=9), 4, 9, 96
    g = torch.Generator().manual_seed(1)
    V = net.cfg.vocab_size
    cache = net.new_cache(b, cap, own_positions=True)
    alone = [net.new_cache(1, cap) for _ in range(b)]
    tokens_in = torch.randint(0, V, (b,), generator=g, dtype=torch.int32)
    lengths = [0] * b
    for step in range(5):
        parents = trees(b, t, step, "random")
        counts = ints([t, 0 if step == 2 else 3, max(1, t - step), t])
        tokens = torch.randint(0, V, (b, t), generator=g, dtype=torch.int32)
        tokens[:, 0] = tokens_in
        # a look ahead, so that some of the guesses are right
        for _ in range(3):
            best = net.argmax(net.forward_tree(*dev(tokens, parents), cache, counts.cuda()).view(b * t, V)).view(b, t).cpu()
            for s in range(b):
                for n in range(1, t):
                    if (n + s) % 3:
                        tokens[s, n] = best[s, parents[s, n]]
        logits = net.forward_tree(*dev(tokens, parents), cache, counts.cuda())
        best = net.argmax(logits.view(b * t, V)).view(b, t).cpu()
        path, count, after = net.decode_tree(*dev(tokens, parents), cache, counts.cuda())
        for s in range(b):
            want, last = walk(tokens[s], parents[s], best[s], int(counts[s]))
            assert path[s].tolist() == want + [-1] * (t - len(want)) and int(after[s]) == last
            for n in want:
                row = net.forward(tokens[s, n:n + 1].cuda(), alone[s])[0]
                assert near(logits[s, n], row)
            lengths[s] += len(want)
            if want:
                tokens_in[s] = last
            k, v = cache.k[:, s, :, :lengths[s]].float(), cache.v[:, s, :, :lengths[s]].float()
            ka, va = alone[s].k[:, 0, :, :lengths[s]].float(), alone[s].v[:, 0, :, :lengths[s]].float()
            assert float((k - ka).abs().max()) <= 0.02 * float(ka.abs().max()) and float((v - va).abs().max()) <= 0.02 * float(va.abs().max())
        assert cache.lens() == lengths and max(lengths) <= cache.host_len <= cap
    assert max(lengths) > 8  # guesses were accepted
    # the sequences go on one token at a time from where they are
    row = net.forward(tokens_in.cuda(), cache)
    for s in range(b):
        assert near(row[s], net.forward(tokens_in[s:s + 1].cuda(), alone[s])[0])
    assert cache.lens() == [n + 1 for n in lengths]
    ctx.check_device_error()


def test_a_recorded_step_with_drafts(ctx):
    """Two recorded steps of two models' caches replayed in turn do what eager steps do; they share no work buffer."""
    import torch
    nets = [small(ctx, seed=4), small(ctx, seed=5, heads=8, kv=2)]
    b, t = 2, 6
    runs = []
    for i, net in enumerate(nets):
        tokens, parents = torch.randint(0, net.cfg.vocab_size, (b, t), dtype=torch.int32).cuda(), trees(b, t, i, "random").cuda()
        eager, recorded = net.new_cache(b, 64, own_positions=True), net.new_cache(b, 64, own_positions=True)
        net.decode_tree(tokens, parents, recorded)                                          # warm
        recorded.pos.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = net.decode_tree(tokens, parents, recorded)
        recorded.pos.zero_()
        runs.append((net, tokens, parents, eager, recorded, graph, got))
    for _ in range(4):
        for net, tokens, parents, eager, recorded, graph, got in runs:
            graph.replay()
        for net, tokens, parents, eager, recorded, graph, got in runs:
            want = net.decode_tree(tokens, parents, eager)
            assert all(torch.equal(a, w) for a, w in zip(got, want)) and torch.equal(eager.pos, recorded.pos)
            n = eager.len
            assert torch.equal(eager.k[:, :, :, :n], recorded.k[:, :, :, :n])
    ctx.check_device_error()


def test_a_full_cache_and_wrong_arguments_are_refused(ctx):
    import torch
    net = small(ctx, max_pos=16)
    cache = net.new_cache(1, 16)
    tokens, parents = torch.zeros(1, 5, dtype=torch.int32, device="cuda"), trees(1, 5, 0, "chain").cuda()
    for _ in range(3):  # five drafts fit where at least five positions are free, however few were accepted
        net.forward_tree(tokens, parents, cache)
        net.accept_tree(cache, *dev(ints([[0, -1, -1, -1, -1]]), ints([1])))
    assert cache.lens() == [3] and cache.host_len == 15
    net.forward_tree(tokens, parents, cache)          # the bound is looked up: 3 are used
    assert cache.host_len == 3
    for _ in range(9):
        net.forward(tokens[:, 0], cache)
    with pytest.raises(ValueError, match="full"):
        net.forward_tree(tokens, parents, cache)
    with pytest.raises(ValueError, match="own"):
        net.forward_tree(tokens.repeat(2, 1), parents.repeat(2, 1), net.new_cache(2, 16))
    with pytest.raises(ValueError):
        net.forward_tree(tokens[:, :4], parents, net.new_cache(1, 16))
    with pytest.raises(ValueError):
        net.forward_tree(tokens.repeat(2, 1), parents.repeat(2, 1), net.new_cache(1, 16))
    ctx.check_device_error()


def test_calls_on_two_streams_at_once(ctx):
    import torch
    from lemonade_burn_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    sets = []
    for b, t, nh, kvh, length, dtype in ((2, 5, 20, 5, 3000, torch.float32), (1, 60, 8, 8, 5000, torch.bfloat16), (3, 30, 4, 1, 900, torch.float32)):
        q = torch.randn(b, t, nh, 128, generator=g, device="cuda").to(dtype)
        k, v = (torch.randn(b, kvh, length + t, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        sets.append((q, k, v, torch.full((b,), length, dtype=torch.int32, device="cuda"), trees(b, t, t).cuda()))
    logits = torch.randn(50, 30000, generator=g, device="cuda")
    want, scored = [ops.attn_tree(*s) for s in sets], ops.token_logprobs(logits, top=9)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(25):
        for s, st, out in zip(sets, streams, got):
            with torch.cuda.stream(st):
                out.append((ops.attn_tree(*s), ops.token_logprobs(logits, top=9)))
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        for a, lp in out:
            assert torch.equal(a, w) and all(torch.equal(x, y) for x, y in zip(lp, scored))
    ctx.check_device_error()


# ---- scores -----------------------------------------------------------------------------------

def check_scores(net, toks, top, want_logits, targets, scale=1.0, got=None):
    lp = want_logits.astype(np.float64) * scale
    lp -= lp.max(-1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(-1, keepdims=True))
    n, V = lp.shape
    slack = 2.0 ** -21 * (math.log(V) + 4) + (V / 256 + 32) * 2.0 ** -24  # as the operator's own test has it
    for i in range(n):
        if targets[i] < 0:
            assert math.isnan(got.logprobs[i])
        else:
            assert abs(got.logprobs[i] - lp[i, targets[i]]) <= slack + 2.0 ** -22 * abs(lp[i, targets[i]])
    assert np.abs(got.entropy + (np.exp(lp) * lp).sum(-1)).max() <= slack * (math.log(V) + 2)
    order = np.argsort(-want_logits, axis=-1, kind="stable")[:, :top]
    assert np.array_equal(got.top_ids, order)
    assert np.abs(got.top_logprobs - np.take_along_axis(lp, order, -1)).max(initial=0) <= slack + 2.0 ** -22 * 40


@pytest.fixture(scope="module")
def families(ctx, tmp_path_factory):
    from lemonade_burn_b200 import dugulorn, model, pefolix, runtime
    p = pefolix.make_config(203, 104, [pefolix.attention_layer(6, 2, 24, 40, 19, 3, 0.9, pefolix.dense_mlp(168)), pefolix.attention_layer(5, 1, 48, 56, 33, 40, 0.5, pefolix.moe_mlp(11, 4, 72, 56))], eps=3e-4)
    d = dugulorn.make_config(203, 104, [dugulorn.delta_layer(6, 3, 24, 20, 4, 72), dugulorn.lightning_layer(3, 18, 44, [0.2, 0.95, 0.9995], None)], eps=3e-4)
    out = {}
    for name, mod, cfg in (("pefolix", pefolix, p), ("dugulorn", dugulorn, d)):
        at = tmp_path_factory.mktemp(name)
        mod.save_checkpoint(at, cfg, mod.random_checkpoint(cfg, 3))
        out[name] = runtime.load_model(at, ctx)
    cfg = model.Config(512, 768, 4, 1, 2, 1003, 1e-5, 500000.0, 400)
    at = tmp_path_factory.mktemp("bitnet")
    model.save_checkpoint(at, cfg, model.random_checkpoint(cfg, 3))
    out["bitnet"] = runtime.load_model(at, ctx)
    return out


@pytest.mark.parametrize("name", ["bitnet", "pefolix", "dugulorn"])
@pytest.mark.parametrize("n,top", [(1, 3), (5, 0), (300, 20)])
def test_scores(families, name, n, top):
    net = families[name]
    V = net.cfg.vocab_size
    rng = np.random.default_rng(n)
    toks, targets = (rng.integers(0, V, n).astype(np.uint32) for _ in range(2))
    cache, plain = net.new_cache(2, 310), net.new_cache(2, 310)
    for seq, given in ((0, None), (1, targets)):
        head = rng.integers(0, V, 4).astype(np.uint32)
        net.forward_rows(head, cache, [], seq=seq), net.forward_rows(head, plain, [], seq=seq)
        want = net.forward_rows(toks, plain, list(range(n)), seq=seq)
        got = net.score(toks, cache, given, top, seq=seq, scale=1.0 if seq else 0.7)
        check_scores(net, toks, top, want, [int(t) for t in (list(toks[1:]) + [-1] if given is None else given)], 1.0 if seq else 0.7, got)
        after = rng.integers(0, V, 2).astype(np.uint32)  # the cache goes on behind the scored tokens
        assert np.array_equal(net.forward_rows(after, cache, [1], seq=seq), net.forward_rows(after, plain, [1], seq=seq))


def test_scores_in_passes_and_refusals(families):
    from lemonade_burn_b200 import _lib
    net = families["bitnet"]
    toks = np.random.default_rng(0).integers(0, 1003, 40).astype(np.uint32)
    whole = net.score(toks, net.new_cache(1, 64), top=4)
    net.set_prefill_rows(7)
    parts = net.score(toks, net.new_cache(1, 64), top=4)
    net.set_prefill_rows(4096)
    # other tiles of the same sums: the logits' own bar
    assert np.abs(parts.logprobs[:-1] - whole.logprobs[:-1]).max() < 0.05 and math.isnan(parts.logprobs[-1])
    cache = net.new_cache(1, 16)
    for bad in (lambda: net.score(toks, cache), lambda: net.score([1003], cache), lambda: net.score([1], cache, targets=[1003]), lambda: net.score([1], cache, seq=1),
                lambda: net.score([1], cache, scale=0.0), lambda: net.score([1], cache, top=33)):
        with pytest.raises(_lib.LbkError):
            bad()
    with pytest.raises(ValueError):
        net.score([1, 2], cache, targets=[1])
    assert net.cache_len(cache) == 0 and net.score([], cache).logprobs.shape == (0,)
    assert net.score(toks[:16], cache).logprobs.shape == (16,) and net.cache_len(cache) == 16


def test_scores_from_the_command_line(families, ctx, tmp_path, capsys):
    from lemonade_burn_b200 import generate, model
    cfg = model.Config(256, 384, 2, 1, 1, 300, 1e-5, 500000.0, 64)
    model.save_checkpoint(tmp_path, cfg, model.random_checkpoint(cfg, 8))
    assert generate.main(["--model", str(tmp_path), "--score", "--prompt", "5,17,3", "--prompt", "9"]) == 0
    lines = capsys.readouterr().out.split("\n")
    net = model.NativeBitNet(tmp_path, ctx)
    want = net.score([5, 17, 3], net.new_cache(1, 8)).logprobs
    assert [float(x) for x in lines[0].split(",")] == pytest.approx(want[:2].tolist(), abs=1e-5) and lines[1] == ""


def test_the_largest_pass(ctx):
    """256 sequences of 128 nodes, 32768 rows: each sequence as it is in a pass by itself."""
    import torch
    net = small(ctx, layers=1, max_pos=140)
    b, t, V = 256, 128, net.cfg.vocab_size
    tokens, parents = dev(torch.randint(0, V, (b, t), generator=torch.Generator().manual_seed(5), dtype=torch.int32), trees(b, t, 5, "random"))
    cache = net.new_cache(b, 140, own_positions=True)
    logits = net.forward_tree(tokens, parents, cache)
    for s in (0, 130, 255):
        alone = net.forward_tree(tokens[s:s + 1].contiguous(), parents[s:s + 1].contiguous(), net.new_cache(1, 140))
        assert near(logits[s], alone[0])
    path, count, after = net.decode_tree(tokens, parents, cache)
    best = net.argmax(logits[255])
    want, last = walk(tokens[255].tolist(), parents[255].tolist(), best.tolist(), t)
    assert count[255].item() == len(want) and path[255, :len(want)].tolist() == want and after[255].item() == last
    ctx.check_device_error()
