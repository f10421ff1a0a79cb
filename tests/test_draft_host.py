"""What the calls around drafted tokens refuse before anything is launched (no GPU needed)."""
import pytest
import torch


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _tree_args(b=2, t=3, kvh=1, cap=8, hd=128, nh=2):
    c = lambda: torch.zeros(b, kvh, cap, hd, dtype=torch.bfloat16)  # noqa: E731
    return dict(q=torch.zeros(b, t, nh * hd), k=torch.zeros(b, t, kvh * hd), v=torch.zeros(b, t, kvh * hd), cos=torch.zeros(cap, hd), sin=torch.zeros(cap, hd), pos=_i(b),
                parents=_i(b, t), kcache=c(), vcache=c(), counts=_i(b))


@pytest.mark.parametrize("change,error", [
    (dict(parents=_i(2)), ValueError), (dict(parents=_i(2, 0)), ValueError), (dict(parents=_i(2, 129)), ValueError), (dict(parents=_i(2, 3).long()), TypeError),
    (dict(pos=_i(1)), ValueError), (dict(pos=_i(2).long()), ValueError), (dict(counts=_i(3)), ValueError), (dict(q=torch.zeros(2, 3, 256).half()), TypeError),
    (dict(q=torch.zeros(2, 3, 250)), ValueError), (dict(k=torch.zeros(2, 3, 256)), ValueError), (dict(kcache=torch.zeros(2, 1, 8, 128)), TypeError),
    (dict(kcache=torch.zeros(3, 1, 8, 128, dtype=torch.bfloat16)), ValueError), (dict(cos=torch.zeros(7, 128)), ValueError), (dict(), ValueError)])
def test_append_refuses(change, error):
    from lemonade_burn_b200 import ops
    with pytest.raises(error if change else (ValueError, RuntimeError)):  # without a change: the tensors are not on a GPU
        ops.rope_kv_append_tree(**{**_tree_args(), **change})


@pytest.mark.parametrize("args,error", [((_i(2, 3), _i(2, 4), _i(2, 4)), ValueError), ((_i(2, 4), _i(2, 4), _i(2, 4).float()), TypeError),
                                        ((_i(2, 4), _i(8), _i(2, 4)), ValueError), ((_i(2, 200), _i(2, 200), _i(2, 200)), ValueError)])
def test_accept_refuses(args, error):
    from lemonade_burn_b200 import ops
    with pytest.raises(error):
        ops.tree_accept(*args)


def test_keep_and_advance_refuse():
    from lemonade_burn_b200 import ops
    c = lambda b: torch.zeros(3, b, 1, 8, 128, dtype=torch.bfloat16)  # noqa: E731
    for args, error in (((c(2), c(3), _i(2), _i(2, 4), _i(2)), ValueError), ((c(2), c(2), _i(2), _i(3, 4), _i(2)), ValueError), ((c(2), c(2).float(), _i(2), _i(2, 4), _i(2)), TypeError),
                        ((c(2)[0], c(2)[0], _i(2), _i(2, 4), _i(2)), ValueError), ((c(2), c(2), _i(3), _i(2, 4), _i(2)), ValueError)):
        with pytest.raises(error):
            ops.kv_keep_path(*args)
    with pytest.raises(ValueError):
        ops.advance_pos_by(_i(2), _i(3))


@pytest.mark.parametrize("logits,tokens,top", [
    (torch.zeros(3, 5, dtype=torch.float64), None, 1), (torch.zeros(3), None, 1), (torch.zeros(3, 0), None, 0), (torch.zeros(3, 5), None, 6), (torch.zeros(3, 50), None, 33),
    (torch.zeros(3, 5), None, -1), (torch.zeros(3, 5), _i(2), 1), (torch.zeros(3, 5), _i(3).long(), 1), (torch.zeros(5, 3).T, None, 1),
    (torch.zeros(5).expand(3, 5), None, 1)])
def test_logprobs_refuse(logits, tokens, top):
    from lemonade_burn_b200 import ops
    with pytest.raises((TypeError, ValueError)):
        ops.token_logprobs(logits, tokens, top)


def test_calls_without_a_context_return_a_status():
    from lemonade_burn_b200 import _lib, build
    build.build()
    lib = _lib.load()
    assert lib.lbk_rope_kv_append_tree(*[None] * 9, 1, 1, 1, 1, 128, 8, None, None, None) == 1
    assert lib.lbk_tree_accept(*[None] * 5, 1, 1, None, None, None, None) == 1
    assert lib.lbk_kv_keep_path(None, None, None, 1, 1024, 1, 1, 128, 8, None, None, None, 1, None) == 1
    assert lib.lbk_advance_pos_by(None, None, None, 1, None) == 1
    assert lib.lbk_token_logprobs(None, 0, None, 5, 1, 5, None, 0, 1.0, 0, None, None, None, None, None) == 1
    assert b"context" in lib.lbk_last_error()
    assert lib.lbk_attn_tree(None, 1, None, 0, *[None] * 5, 1, 1, 1, 1, 128, 8, 1.0, None, None, 0, None) == 1
    assert lib.lbk_attn_tree_scratch(None, 1, 1, 1) == 0
    assert lib.lbk_model_score(None, None, 0, None, 0, None, 1.0, 0, None, None, None, None) == 1


def test_a_missing_extension_module_is_an_error(monkeypatch, tmp_path):
    from lemonade_burn_b200 import _lib, ops
    monkeypatch.setattr(ops, "_native", None)
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "liblbk.so")
    with pytest.raises(RuntimeError, match="missing"):
        ops.advance_pos_by(_i(1), _i(1))


def test_a_model_refuses_drafts_before_anything_is_launched():
    from types import SimpleNamespace

    from lemonade_burn_b200.model import BitNet
    net = SimpleNamespace(cfg=SimpleNamespace(head_dim=lambda: 128), final_norm=SimpleNamespace(device=torch.device("cuda:0")))
    there = lambda *shape: SimpleNamespace(dtype=torch.int32, shape=torch.Size(shape), dim=lambda: len(shape), device=torch.device("cuda:0"))  # noqa: E731
    cache = SimpleNamespace(b=2, own_positions=True, pos=there(2))
    refused = [(_i(2, 3), _i(2, 3), None), (there(2, 3), _i(2, 3), None), (_i(2, 3), there(2, 3), None), (there(2, 3), there(2, 3), _i(2)), (there(2, 0), there(2, 0), None),
               (there(2, 129), there(2, 129), None), (there(3, 3), there(3, 3), None), (there(2, 3), there(2, 4), None), (_i(2, 3).long(), _i(2, 3), None)]
    for tokens, parents, counts in refused:
        with pytest.raises(ValueError):
            BitNet.forward_tree(net, tokens, parents, cache, counts)
    with pytest.raises(ValueError, match="live on"):
        BitNet.forward_tree(net, there(2, 3), there(2, 3), SimpleNamespace(b=2, own_positions=True, pos=_i(2)))


def test_a_part_of_the_library_has_some_of_the_calls():
    """A process that serves one family may load that family's part: it has log probabilities, but no trees."""
    import subprocess
    import sys
    code = """
import types, torch
from lemonade_burn_b200 import _lib, build, ops
build.build()
whole = _lib.load()
_lib._lib = types.SimpleNamespace(lbk_token_logprobs=whole.lbk_token_logprobs)
ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)
for call in (lambda: ops.advance_pos_by(ints(1), ints(1)), lambda: ops.tree_accept(ints(1, 1), ints(1, 1), ints(1, 1)), lambda: ops.token_logprobs(torch.zeros(2))):
    try:
        call()
    except Exception as e:
        print(type(e).__name__, e)
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert out.stdout.splitlines() == ["RuntimeError the library that is loaded has no lbk_advance_pos_by", "RuntimeError the library that is loaded has no lbk_tree_accept",
                                       "ValueError logits are [rows, vocab]"]


def test_keep_that_advances_refuses():
    from lemonade_burn_b200 import _lib, build, ops
    build.build()
    c = torch.zeros(3, 2, 1, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.kv_keep_path(c, c, _i(2), _i(3, 4), _i(2), advance=True)
    assert _lib.load().lbk_advance_pos_path(None, None, None, None, 1, 1, 8, None) == 1


def test_rows_of_nodes_without_a_context():
    from lemonade_burn_b200 import _lib, build
    build.build()
    assert _lib.load().lbk_embed_tree_bf16(None, None, 5, None, None, 1, 1, 8, None, None) == 1


def test_scores_of_many_prompts_take_one_cache(monkeypatch, capsys):
    """The command's prompts come one behind the other: one cache, as long as the longest, serves them."""
    from types import SimpleNamespace

    import numpy as np

    from lemonade_burn_b200 import _lib, build, generate, runtime
    made, used = [], []

    class Net:
        def new_cache(self, b, cap):
            made.append((b, cap))
            return SimpleNamespace(free=cap)

        def reset_cache(self, cache):
            cache.free = made[0][1]

        def score(self, prompt, cache):
            cache.free -= len(prompt)
            used.append(cache.free)
            return SimpleNamespace(logprobs=np.arange(len(prompt), dtype=np.float32))

        def close(self):
            pass
    monkeypatch.setattr(_lib, "use", lambda path: None)
    monkeypatch.setattr(build, "library_for", lambda architecture: None)
    monkeypatch.setattr(runtime, "architecture_of", lambda directory: "")
    monkeypatch.setattr(runtime, "load_model", lambda directory, dtype: Net())
    assert generate.main(["--model", "x", "--score", "--prompt", "1,2", "--prompt", "3,4,5,6", "--prompt", "7"]) == 0
    assert made == [(1, 4)] and used == [2, 0, 3]
    assert capsys.readouterr().out.splitlines() == ["0.000000", "0.000000,1.000000,2.000000", ""]
