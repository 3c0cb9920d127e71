"""PagedPath (many requests over the paged 8-bit KV cache) on small models
against MatrixPath.prompt_step, whose f16 cache and attention repeat the
reference's arithmetic.

The cache's rounding is at most half a step of each block's largest magnitude
(1 / 254 of it, some 0.8 % of a normal value's size in the mean square), the
attention averages it, and three layers add three of them to a residual stream
the norms keep at unit size: the logits agree within 5 % of their norm."""

from __future__ import annotations

import numpy as np
import pytest

from siphon_b200 import quant as Q
from siphon_b200 import synth_model as sm

pytestmark = pytest.mark.gpu


def alone(sicu, path, sh, tokens):
    """Every token's logits from the one-sequence path."""
    import torch
    from siphon_b200 import model_path as mp
    m = mp.MatrixPath(sicu, sh, torch.device("cuda", 0), embed=True, n_ctx=256, gguf_path=path,
                      max_tokens=max(2, len(tokens)))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    m.tokens[:len(tokens)].copy_(torch.tensor(tokens))
    torch.cuda.synchronize()
    m.prompt_step(st, len(tokens))
    st.synchronize()
    out = m.y["head"][:len(tokens)].cpu().numpy().astype(np.float64)
    m.close()
    return out


@pytest.mark.parametrize("sh", [sm.SMALL, sm.SMALL_QWEN], ids=["llama", "qwen2"])
def test_requests_in_one_batch_match_each_alone(sicu, tmp_path, sh):
    import torch
    from siphon_b200.serving import PagedPath
    path = sm.write_llama(tmp_path / "m.gguf", sh, seed=7, wtype=Q.Q8_0)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, sh.n_vocab, n).tolist() for n in (45, 1, 17, 70)]
    p = PagedPath(sicu, sh, torch.device("cuda", 0), max_seqs=5, max_len=128, n_pages=24, page=16, max_tokens=160,
                  gguf_path=path)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()

    def close(row, want):
        got = p.y["head"][row].cpu().numpy().astype(np.float64)
        assert np.linalg.norm(got - want) <= 0.05 * np.linalg.norm(want)

    # the first 40 tokens of the longest prompt, then its rest beside three others
    p.step(st, [0, 0, 0, 40, 0], prompts[3][:40])
    p.step(st, [45, 1, 17, 30, 0], prompts[0] + prompts[1] + prompts[2] + prompts[3][40:])
    st.synchronize()
    seqs = [list(t) for t in prompts]
    for i in range(4):
        close(i, alone(sicu, path, sh, seqs[i])[-1])
    # greedy steps, one request ending on the way and another taking its place
    for k in range(12):
        choice = p.next.cpu().tolist()
        live = [i for i, n in enumerate(p.len_host) if n]
        for i in live:
            seqs[i].append(choice[i])
        p.decode(st)
        st.synchronize()
        if k in (0, 5, 11):
            for row, i in enumerate(live):
                close(row, alone(sicu, path, sh, seqs[i])[-1])
        if k == 5:
            free = int(p.n_free.cpu()[0])
            gone = -(-p.len_host[2] // 16)
            p.retire(st, [2])
            st.synchronize()
            assert int(p.n_free.cpu()[0]) == free + gone
            seqs[2] = rng.integers(0, sh.n_vocab, 9).tolist()
            p.step(st, [0, 0, 9, 0, 0], seqs[2])
            st.synchronize()
            close(0, alone(sicu, path, sh, seqs[2])[-1])
    assert sicu.status() == 0
    held = sum(-(-n // 16) for n in p.len_host)
    assert int(p.n_free.cpu()[0]) == 24 - held
    used = [p.table[i, :-(-n // 16)].cpu().tolist() for i, n in enumerate(p.len_host)]
    pages = sum(used, []) + p.free[:24 - held].cpu().tolist()
    assert sorted(pages) == list(range(24))                  # every page owned once or free
    p.close()
