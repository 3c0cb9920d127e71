"""The host side of PagedPath on the CPU, with a recording stand-in for the
CUDA library: the order of the library calls, the sizes a step passes, and its
argument errors. The numerics are the GPU tests'."""

from __future__ import annotations

import inspect

import pytest

from siphon_b200 import lib
from siphon_b200 import serving
from siphon_b200 import synth_model as sm


class _Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        sig = inspect.signature(getattr(lib.SiphonCuda, name))

        def call(*a, **k):
            b = sig.bind(None, *a, **k)
            self.calls.append((name, b.arguments))
            return 4096 if name in ("prefill_pack_bytes", "kv8_attention_ws") else None
        return call


class _Stream:
    cuda_stream = None


def make(tmp_path, sh=sm.SMALL, **kw):
    import torch
    path = sm.write_llama(tmp_path / "m.gguf", sh, seed=3)
    rec = _Recorder()
    a = dict(max_seqs=3, max_len=64, n_pages=9, page=16, max_tokens=40, gguf_path=path)
    a.update(kw)
    p = serving.PagedPath(rec, sh, torch.device("cpu"), **a)
    rec.calls.clear()
    return p, rec


def test_step_call_order_and_sizes(tmp_path):
    p, rec = make(tmp_path)
    n = p.step(_Stream(), [5, 0, 20], list(range(25)))
    names = [c[0] for c in rec.calls]
    assert n == len(rec.calls)
    assert names[:3] == ["kv8_plan", "kv8_attention_ws", "row_to_f32_dev"] and names[-1] == "argmax"
    for il in range(sm.SMALL.n_layer):
        assert names.count("kv8_store") == names.count("kv8_attention") == sm.SMALL.n_layer
    stores = [i for i, c in enumerate(names) if c == "kv8_store"]
    assert all(names[i + 1] == "kv8_attention" and names[i - 1].startswith("gemm_prefill") for i in stores)
    plan = rec.calls[0][1]
    assert plan["n_tok"] == 25 and plan["max_pages"] == 4 and plan["n_free"] is plan["n_free_out"]
    attn = rec.calls[stores[0] + 1][1]["attn"]
    assert (attn.n_tok, attn.max_new, attn.max_len, attn.n_seq, attn.n_head) == (25, 20, 20, 3, 8)
    assert rec.calls[-1][1]["m"] == 2                        # two requests advanced
    rec.calls.clear()
    p.decode(_Stream())
    attn = [c for c in rec.calls if c[0] == "kv8_attention"][0][1]["attn"]
    assert (attn.n_tok, attn.max_new, attn.max_len) == (2, 1, 21) and p.len_host == [6, 0, 21]
    p.retire(_Stream(), [2])
    assert rec.calls[-1][0] == "kv8_release" and p.len_host == [6, 0, 0]


def test_step_qwen2_bias_adds(tmp_path):
    p, rec = make(tmp_path, sm.SMALL_QWEN)
    p.step(_Stream(), [3, 3, 3], list(range(9)))
    names = [c[0] for c in rec.calls]
    assert names.count("add_bias") == 3 * sm.SMALL_QWEN.n_layer
    assert p.rope.neox == 1


def test_step_argument_errors(tmp_path):
    p, rec = make(tmp_path)
    for fresh, tokens in (([41, 0, 0], range(41)), ([0, 0, 0], []), ([1, 1], [1, 2]), ([2, 0, 0], [1]), ([3, -1, 0], [1, 2])):
        with pytest.raises(ValueError):
            p.step(_Stream(), fresh, list(tokens))
    p.step(_Stream(), [40, 0, 0], list(range(40)))
    with pytest.raises(ValueError, match="past 64"):
        p.step(_Stream(), [25, 0, 0], list(range(25)))
    q, _ = make(tmp_path, n_pages=3)
    with pytest.raises(ValueError, match="pages"):
        q.step(_Stream(), [17, 17, 0], list(range(34)))
    with pytest.raises(ValueError, match="no request"):
        q.decode(_Stream())


@pytest.mark.parametrize("requests", [[0, 3], [-1], [1, -3]])
def test_retire_refuses_places_it_does_not_have(tmp_path, requests):
    p, rec = make(tmp_path)
    p.step(_Stream(), [5, 1, 20], list(range(26)))
    rec.calls.clear()
    with pytest.raises(ValueError):
        p.retire(_Stream(), requests)
    assert not rec.calls and p.len_host == [5, 1, 20]
