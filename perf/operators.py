"""The paged 8-bit KV cache's operators as cases to measure: block tables and
slot maps from request lengths (kv8_plan), the quantizing store of new tokens
with RoPE and the read-back of stored rows (kv8_store, kv8_load), and
attention over the cache (kv8_attention) for single tokens and for prompts.

Cache layout, one layer: codes int8 [n_pages][n_head_kv][page][head_dim] for
K and V, one f32 scale per 16-token block and KV head
[n_pages][n_head_kv][page / 16]; a stored value is code * scale.

Where ``own`` is false, run() computes in plain f32 torch operations; where it
is true it calls the library.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BLOCK = 16                     # tokens per quantization block

# query heads, KV heads, head size, half-split RoPE pairs, RoPE base
SHAPES = {
    "tinyllama": (32, 4, 64, False, 10000.0),
    "llama3-8b": (32, 8, 128, False, 500000.0),
    "qwen2.5-32b": (40, 8, 128, True, 1000000.0),
    "small": (8, 2, 64, False, 10000.0),
    "ungrouped": (12, 12, 64, True, 10000.0),
    "one-kv-head": (16, 1, 128, False, 10000.0),
    "head-96": (24, 8, 96, True, 10000.0),
    "head-256": (8, 4, 256, True, 10000.0),
}


# ---- the cases -------------------------------------------------------------------

def _plan(name, **kw):
    c = {"op": "plan", "lens": 1, "page": 16, "n_seq": 1, "past_lo": 0, "past_hi": 0, "new_lo": 1, "new_hi": 1,
         "idle": 0, **kw}
    return {**c, **({"name": name} if name else {})}


def _store(name, **kw):
    c = {"op": "store", "shape": "tinyllama", "type": "f32", "lens": 1, "page": 16, "n_seq": 1, "past_lo": 0,
         "past_hi": 0, "new_lo": 1, "new_hi": 1, "idle": 0, "rope": True, **kw}
    return {**c, **({"name": name} if name else {})}


def _attn(name, **kw):
    c = {"op": "attention", "shape": "tinyllama", "type": "f32", "lens": 1, "page": 16, "n_seq": 1, "past_lo": 0,
         "past_hi": 0, "new_lo": 1, "new_hi": 1, "idle": 0, "rope": True, "cap": 0.0, "slopes": False, "window": 0,
         "prefix": False, "first": False, **kw}
    return {**c, **({"name": name} if name else {})}


def listed():
    return [
        # a decode step of 64 running requests: one new page here and there; latency is all of it
        _plan("plan_decode_64", n_seq=64, past_lo=1, past_hi=2047, lens=11),
        # a busy server's step: 2048 requests, most decoding or idle, the others with
        # chunks of prompts of up to 128 tokens (some 60,000 tokens in all)
        _plan("plan_step_2048", n_seq=2048, past_lo=0, past_hi=2000, new_lo=1, new_hi=128, idle=300, page=32, lens=12),
        # one token each of 8 sequences at the TinyLlama shape (the decode batch limit of the products)
        _store("store_decode_8", n_seq=8, past_lo=1, past_hi=511, lens=13),
        # ragged prompts of 7 requests at the Llama-3-8B shape, two of them continued mid-block
        _store("store_prompts_7", shape="llama3-8b", n_seq=7, past_lo=0, past_hi=100, new_lo=500, new_hi=4096, page=64,
               lens=14),
        # the smallest decode batch: 8 TinyLlama-shape sequences below the benchmark's context
        _attn("decode_tinyllama_8", n_seq=8, past_lo=0, past_hi=511, lens=15),
        # an ordinary serving step: 64 Llama-3-8B-shape sequences of 500 to 8000 tokens, one slot idle
        _attn("decode_llama_64", shape="llama3-8b", n_seq=64, past_lo=500, past_hi=8000, idle=1, page=32, lens=16),
        # one long document: a single Qwen2.5-32B-shape sequence past 128K tokens, f16 activations
        _attn("decode_long_1", shape="qwen2.5-32b", type="f16", n_seq=1, past_lo=131075, past_hi=131075, page=64, lens=17),
        # models with capped scores, distance bias and a sliding window; evicted starts
        _attn("decode_masked_48", shape="llama3-8b", type="f16", n_seq=48, past_lo=0, past_hi=4000, cap=50.0,
              slopes=True, window=1024, first=True, lens=18),
        # the benchmark's 512-token TinyLlama-shape prompt
        _attn("prompt_tinyllama_512", n_seq=1, new_lo=512, new_hi=512, lens=19),
        # a long prompt at the Llama-3-8B shape, f16 activations; odd length
        _attn("prompt_llama_8k", shape="llama3-8b", type="f16", n_seq=1, new_lo=8191, new_hi=8191, page=64, lens=20),
        # a step that mixes chunks of prompts with cached prefixes, short tails and
        # an idle slot at the Qwen2.5-32B shape, f32, bidirectional prefixes, evicted starts
        _attn("prompt_mixed_6", shape="qwen2.5-32b", n_seq=6, past_lo=0, past_hi=3001, new_lo=1, new_hi=1501, idle=1,
              prefix=True, first=True, page=32, lens=21),
        # two prompts of a model with capped scores, distance bias and a window
        _attn("prompt_capped_2", shape="llama3-8b", type="f16", n_seq=2, new_lo=4001, new_hi=6000, cap=30.0,
              slopes=True, window=2048, page=128, lens=22),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page = rng.choice((16, 32, 64, 128))
    lens = rng.randrange(1 << 30)
    kind = rng.choice(("plan", "store", "decode", "decode", "prompt", "prompt"))
    if kind == "plan":
        n_seq = _log_int(rng, 1, 2048)
        return _plan(None, n_seq=n_seq, page=page, lens=lens, past_lo=0, past_hi=_log_int(rng, 16, 8192),
                     new_lo=rng.choice((0, 1)), new_hi=rng.choice((1, _log_int(rng, 2, 1000))),
                     idle=rng.randrange(0, n_seq // 4 + 1))
    shape = rng.choice(tuple(SHAPES))
    typ = rng.choice(("f32", "f16"))
    rope = rng.random() < 0.8
    if kind == "store":
        n_seq = _log_int(rng, 1, 256)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(3, 16384 // n_seq))
        return _store(None, shape=shape, type=typ, rope=rope, n_seq=n_seq, page=page, lens=lens, past_lo=0,
                      past_hi=_log_int(rng, 1, 2048), new_lo=min(new, rng.choice((1, new))), new_hi=new)
    masks = dict(cap=rng.choice((0.0, 0.0, 20.0, 50.0)), slopes=rng.random() < 0.3, prefix=rng.random() < 0.25,
                 first=rng.random() < 0.25, window=rng.choice((0, 0, 0, _log_int(rng, 1, 4096))))
    hkv, hd = SHAPES[shape][1:3]
    if kind == "decode":
        n_seq = _log_int(rng, 1, 128)
        # cached elements of K bounded by those of the listed decode batch
        most = min(131072, (1 << 28) // (n_seq * hkv * hd))
        return _attn(None, shape=shape, type=typ, rope=rope, n_seq=n_seq, page=page, lens=lens, past_lo=0,
                     past_hi=_log_int(rng, 1, most), new_lo=1, new_hi=rng.choice((1, 1, 1, rng.randrange(2, 9))),
                     idle=rng.randrange(0, n_seq // 4 + 1), **masks)
    n_seq = _log_int(rng, 1, 12)
    new = _log_int(rng, 9, max(10, 6000 // n_seq))
    return _attn(None, shape=shape, type=typ, rope=rope, n_seq=n_seq, page=page, lens=lens, past_lo=0,
                 past_hi=rng.choice((0, _log_int(rng, 1, 4000))), new_lo=min(new, rng.choice((1, new))), new_hi=new,
                 idle=rng.choice((0, 0, n_seq // 4)), **masks)


# ---- what a case stands for ------------------------------------------------------

def _lengths(c):
    """(past, new) per request; idle requests add nothing."""
    rng = random.Random(c["lens"])
    past = [rng.randint(c["past_lo"], c["past_hi"]) for _ in range(c["n_seq"])]
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["n_seq"])]
    for i in rng.sample(range(c["n_seq"]), c["idle"]):
        new[i] = 0
    if c["op"] == "plan":      # most requests of a server's step decode one token
        for i in range(c["n_seq"]):
            if new[i] > 1 and rng.random() < 0.5:
                new[i] = 1
    if not any(new):
        new[0] = 1
    return past, new


def _mask_arrays(c, past, new):
    """Per-request prefix lengths (positions below them see each other both
    ways) and first visible positions (earlier ones were evicted)."""
    rng = random.Random(c["lens"] + 1)
    total = [p + n for p, n in zip(past, new)]
    prefix = [rng.randint(0, t) for t in total]
    # about one request in four lost its oldest tokens; now and then so many
    # that its first new rows see nothing
    first = [0 if rng.random() < 0.75 else rng.randint(0, t) for t in total]
    return prefix, first


def _slopes(n_head):
    return [2.0 ** (-8.0 * (h + 1) / n_head) for h in range(n_head)]


def _seen(c):
    """Sum over requests and rows of the positions a row sees, and over
    requests of the positions any of its rows sees."""
    past, new = _lengths(c)
    prefix, first = _mask_arrays(c, past, new)
    pairs = union = 0
    for i in range(c["n_seq"]):
        if not new[i]:
            continue
        p = np.arange(past[i], past[i] + new[i], dtype=np.int64)
        hi = np.maximum(p + 1, min(prefix[i], past[i] + new[i])) if c["prefix"] else p + 1
        lo = np.maximum(p + 1 - c["window"], 0) if c["window"] else np.zeros_like(p)
        if c["first"]:
            lo = np.maximum(lo, first[i])
        pairs += int(np.maximum(hi - lo, 0).sum())
        union += int(max(hi.max() - lo.min(), 0))
    return pairs, union


def work(c):
    past, new = _lengths(c)
    n_tok = sum(new)
    if c["op"] == "plan":
        fresh_pages = sum(-(-(p + n) // c["page"]) - -(-p // c["page"]) for p, n in zip(past, new))
        return {"bytes": 4 * c["n_seq"] * 4 + 12 * n_tok + 8 * fresh_pages + 8, "flops": 2 * c["n_seq"]}
    n_head, hkv, hd, _, _ = SHAPES[c["shape"]]
    size = 4 if c["type"] == "f32" else 2
    rope = 2 * 4 * (hd // 2) * n_tok if c["rope"] else 0
    if c["op"] == "store":
        blocks = sum(-(-(p + n) // BLOCK) - p // BLOCK for p, n in zip(past, new) if n)
        back = sum(p % BLOCK + n for p, n in zip(past, new) if n)      # rows of the touched blocks, read back
        row = 2 * hkv * hd
        # in: k, v, slots, positions, tables; out: codes and scales; then the touched rows as values
        return {"bytes": n_tok * (row * (size + 1) + 12) + rope + 2 * 4 * hkv * blocks + back * row * (1 + size),
                "flops": n_tok * row * 6}
    pairs, union = _seen(c)
    return {"bytes": 2 * n_tok * n_head * hd * size + rope + union * hkv * (2 * hd + 2 * 4 // BLOCK) + 4 * union // c["page"],
            "flops": 4 * hd * n_head * pairs}


# ---- inputs ----------------------------------------------------------------------

def _dtype(c):
    return torch.float32 if c["type"] == "f32" else torch.float16


def _rope_tables(rows, hd, base, dev):
    theta = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * \
        base ** (-2.0 * torch.arange(hd // 2, device=dev, dtype=torch.float64) / hd)
    return theta.cos().float().contiguous(), theta.sin().float().contiguous()


def _filled(gen, n_pages, hkv, page, hd, channels):
    """A cache part as earlier steps left it: normal values (K with a few
    large channels, as keys have) quantized by block of 16 tokens."""
    codes = torch.empty(n_pages, hkv, page, hd, dtype=torch.int8, device=gen.device)
    scale = torch.empty(n_pages, hkv, page // BLOCK, dtype=torch.float32, device=gen.device)
    step = max(1, (1 << 26) // (hkv * page * hd))
    for a in range(0, n_pages, step):
        b = min(n_pages, a + step)
        x = torch.randn(b - a, hkv, page, hd, device=gen.device, generator=gen) * channels
        x = x.view(b - a, hkv, page // BLOCK, BLOCK * hd)
        s = x.abs().amax(-1) / 127.0
        scale[a:b] = s
        codes[a:b] = torch.round(x / s[..., None]).clamp_(-127, 127).to(torch.int8).view(b - a, hkv, page, hd)
    return codes, scale


def _inputs(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    past, new = _lengths(c)
    total = [p + n for p, n in zip(past, new)]
    page, n_seq, n_tok = c["page"], c["n_seq"], sum(new)
    pages = [-(-t // page) for t in total]
    held = [-(-p // page) for p in past]
    max_pages = max(max(pages), 1)
    n_pages = sum(pages) + 5
    order = torch.randperm(n_pages, device=dev, generator=gen).to(torch.int32)   # a used pool: pages in no order
    i32 = dict(dtype=torch.int32, device=dev)
    st = {"case": c, "past_host": past, "new_host": new, "total_host": total, "n_tok": n_tok, "max_pages": max_pages,
          "n_pages": n_pages, "past": torch.tensor(past, **i32), "new": torch.tensor(new, **i32)}
    rows = torch.repeat_interleave(torch.arange(n_seq), torch.tensor(held if c["op"] == "plan" else pages)).to(dev)
    cols = torch.cat([torch.arange(h) for h in (held if c["op"] == "plan" else pages)]).to(dev)
    table = torch.zeros(n_seq, max_pages, **i32)
    table[rows, cols] = order[:rows.numel()]
    st["table"] = table
    if c["op"] == "plan":
        # the free pages' stack: a buffer for every page of the pool, its first n_free entries valid
        n_free = n_pages - rows.numel()
        st["free"] = torch.cat((order[rows.numel():], torch.zeros(n_pages - n_free, **i32)))
        st["n_free"] = torch.tensor([n_free], **i32)
        return st
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    st["len"], st["cu"] = torch.tensor(total, **i32), torch.tensor(cu, **i32)
    n_head, hkv, hd, neox, base = SHAPES[c["shape"]]
    channels = torch.ones(hkv, 1, hd, device=dev)
    channels[:, :, torch.randperm(hd, device=dev, generator=gen)[:max(1, hd // 32)]] = 6.0
    st["k"], st["k_scale"] = _filled(gen, n_pages, hkv, page, hd, channels)
    st["v"], st["v_scale"] = _filled(gen, n_pages, hkv, page, hd, torch.ones(hkv, 1, hd, device=dev))
    st["rows"] = max_pages * page
    st["cos"], st["sin"] = _rope_tables(st["rows"], hd, base, dev)
    if c["op"] == "store":
        st["dk"] = (torch.randn(n_tok, hkv, hd, device=dev, generator=gen) * channels[:, 0]).to(_dtype(c))
        st["dv"] = torch.randn(n_tok, hkv, hd, device=dev, generator=gen).to(_dtype(c))
        seq = torch.repeat_interleave(torch.arange(n_seq), torch.tensor(new)).to(dev)
        pos = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).to(dev)
        st["slot"] = table[seq, pos // page].long() * page + pos % page
        st["pos"] = pos.to(torch.int32)
        # every valid row of the touched blocks: what the step changed
        bseq = torch.repeat_interleave(torch.arange(n_seq), torch.tensor([p % BLOCK + n if n else 0
                                                                          for p, n in zip(past, new)])).to(dev)
        bpos = torch.cat([torch.arange(p - p % BLOCK, p + n) if n else torch.arange(0)
                          for p, n in zip(past, new)]).to(dev)
        st["back"] = table[bseq, bpos // page].long() * page + bpos % page
        return st
    st["q"] = torch.randn(n_tok, n_head, hd, device=dev, generator=gen).to(_dtype(c))
    prefix, first = _mask_arrays(c, past, new)
    st["prefix_host"], st["first_host"] = prefix, first
    st["prefix"] = torch.tensor(prefix, **i32) if c["prefix"] else None
    st["first"] = torch.tensor(first, **i32) if c["first"] else None
    st["slopes"] = torch.tensor(_slopes(n_head), dtype=torch.float32, device=dev) if c["slopes"] else None
    st["scale"] = float(np.float32(1.0 / math.sqrt(hd)))
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _bind(st)
    return st


# ---- the library's calls ---------------------------------------------------------

def _bind(st):
    """The handle, descriptors, outputs and workspace a program keeps."""
    from siphon_b200 import lib as L
    c = st["case"]
    s = st["lib"] = L.load()
    torch.cuda.init()
    s.init(0)
    dev = st["table"].device
    if c["op"] == "plan":
        i32 = dict(dtype=torch.int32, device=dev)
        st["o_cu"], st["o_len"], st["o_nfree"] = (torch.empty(c["n_seq"] + 1, **i32), torch.empty(c["n_seq"], **i32),
                                                  torch.empty(1, **i32))
        st["o_slot"] = torch.empty(st["n_tok"], dtype=torch.int64, device=dev)
        st["o_pos"] = torch.empty(st["n_tok"], **i32)
        return
    n_head, hkv, hd, neox, _ = SHAPES[c["shape"]]
    st["type"] = L.T_F32 if c["type"] == "f32" else L.T_F16
    st["cache"] = L.kv8_cache(st["k"], st["v"], st["k_scale"], st["v_scale"], st["n_pages"], c["page"], hkv, hd)
    st["rope"] = L.rope(st["cos"], st["sin"], st["rows"], hd, neox) if c["rope"] else None
    if c["op"] == "store":
        st["o_k"] = torch.empty(st["back"].numel(), hkv, hd, dtype=_dtype(c), device=dev)
        st["o_v"] = torch.empty_like(st["o_k"])
        return
    st["out"] = torch.empty_like(st["q"])
    st["attn"] = L.kv8_attn(st["type"], n_head, st["n_tok"], st["table"], st["max_pages"], st["len"], st["cu"],
                            c["n_seq"], max(st["new_host"]), max(st["total_host"]), st["scale"], cap=c["cap"],
                            slopes=st["slopes"], window=c["window"], prefix=st["prefix"], first=st["first"],
                            rope=st["rope"])
    st["ws"] = torch.empty(max(s.kv8_attention_ws(st["cache"], st["attn"]), 1), dtype=torch.uint8, device=dev)


def _run_own(st):
    s, c = st["lib"], st["case"]
    h = torch.cuda.current_stream().cuda_stream
    if c["op"] == "plan":
        s.kv8_plan(st["past"], st["new"], c["n_seq"], c["page"], st["table"], st["max_pages"], st["free"],
                   st["n_pages"], st["n_free"], st["o_nfree"], st["n_tok"], st["o_cu"], st["o_len"], st["o_slot"],
                   st["o_pos"], stream=h)
        return st["table"], st["o_cu"], st["o_len"], st["o_slot"], st["o_pos"], st["o_nfree"]
    if c["op"] == "store":
        s.kv8_store(st["cache"], st["type"], st["dk"], st["dv"], st["slot"], st["n_tok"], pos=st["pos"],
                    rope=st["rope"], stream=h)
        s.kv8_load(st["cache"], st["type"], st["back"], st["back"].numel(), st["o_k"], st["o_v"], stream=h)
        return st["o_k"], st["o_v"]
    s.kv8_attention(st["cache"], st["attn"], st["q"], st["out"], st["ws"], stream=h)
    return st["out"]


# ---- the plain forms -------------------------------------------------------------

def _rotate(x, pos, st):
    """RoPE of rows x [n][heads][hd] (f32) at positions pos [n]."""
    neox = SHAPES[st["case"]["shape"]][3]
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]
    if neox:
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _plain_plan(st):
    c = st["case"]
    past, new, page, free = st["past"].long(), st["new"].long(), c["page"], st["free"]
    dev = past.device
    total = past + new
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=dev), new.cumsum(0)))
    held, need = (past + page - 1) // page, (total + page - 1) // page
    take = need - held
    start = take.cumsum(0) - take
    n = int(take.sum())
    rows = torch.repeat_interleave(torch.arange(c["n_seq"], device=dev), take)
    j = torch.arange(n, device=dev)
    table = st["table"]
    n_free = st["n_free"].long()
    table[rows, held[rows] + j - start[rows]] = free[n_free - 1 - j]      # the stack's top first
    seq = torch.repeat_interleave(torch.arange(c["n_seq"], device=dev), new)
    pos = past[seq] + torch.arange(st["n_tok"], device=dev) - cu[seq]
    slot = table[seq, pos // page].long() * page + pos % page
    return table, cu.int(), total.int(), slot, pos.int(), (n_free - n).int()


def _plain_quantize(x, codes, scale, slot, page):
    """Stores rows x [n][hkv][hd] (f32) at their slots: a block that gets its
    first rows takes their largest magnitude / 127 as scale; one that already
    holds rows keeps the larger of its scale and theirs, its rows requantized."""
    hkv, hd = x.shape[1:]
    block, off = slot // BLOCK, slot % BLOCK
    ids, inv = torch.unique_consecutive(block, return_inverse=True)
    nb = ids.numel()
    amax = torch.zeros(nb, hkv, device=x.device).index_reduce_(0, inv, x.abs().amax(-1), "amax")
    lead = torch.full((nb,), BLOCK, dtype=torch.int64, device=x.device).index_reduce_(0, inv, off, "amin")
    pg, sub = ids // (page // BLOCK), ids % (page // BLOCK)
    cb = codes.view(codes.shape[0], hkv, page // BLOCK, BLOCK, hd)
    before = torch.where((lead > 0)[:, None], scale[pg, :, sub], torch.zeros((), device=x.device))
    s = torch.maximum(before, amax / 127.0)
    r = torch.where(s > 0, 1.0 / s, torch.zeros((), device=x.device))
    held = cb[pg, :, sub].float()
    cb[pg, :, sub] = torch.round(held * (before * r)[:, :, None, None]).to(torch.int8)
    scale[pg, :, sub] = s
    q = torch.round(x * r[inv][:, :, None]).clamp_(-127, 127).to(torch.int8)
    codes[slot // page, :, slot % page] = q


def _plain_store(st):
    c = st["case"]
    page = c["page"]
    k, v = st["dk"].float(), st["dv"].float()
    if c["rope"]:
        k = _rotate(k, st["pos"].long(), st)
    out = []
    for x, codes, scale in ((k, st["k"], st["k_scale"]), (v, st["v"], st["v_scale"])):
        _plain_quantize(x, codes, scale, st["slot"], page)
        b = st["back"]
        pg, off = b // page, b % page
        out.append((codes[pg, :, off].float() * scale[pg, :, off // BLOCK][..., None]).to(_dtype(c)))
    return tuple(out)


def _plain_attention(st):
    c = st["case"]
    n_head, hkv, hd, _, _ = SHAPES[c["shape"]]
    g, page = n_head // hkv, c["page"]
    out = torch.empty_like(st["q"])
    dev = out.device
    at = 0
    for i, (n, total) in enumerate(zip(st["new_host"], st["total_host"])):
        if n == 0:
            continue
        ids = st["table"][i, :-(-total // page)].long()
        kv = []
        for codes, scale in ((st["k"], st["k_scale"]), (st["v"], st["v_scale"])):
            x = codes[ids].float() * torch.repeat_interleave(scale[ids], BLOCK, -1)[..., None]
            kv.append(x.permute(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :total])
        k, v = kv
        j = torch.arange(total, device=dev)
        step = max(1, (1 << 27) // (n_head * total))
        for a in range(0, n, step):
            b = min(n, a + step)
            pos = torch.arange(total - n + a, total - n + b, device=dev)
            q = st["q"][at + a:at + b].float()
            if c["rope"]:
                q = _rotate(q, pos, st)
            q = q.view(b - a, hkv, g, hd).permute(1, 2, 0, 3).reshape(hkv, g * (b - a), hd)
            s = (q @ k.transpose(1, 2)).mul_(st["scale"]).view(hkv, g, b - a, total)
            if c["cap"]:
                s = torch.tanh(s / c["cap"]) * c["cap"]
            d = pos[:, None] - j
            if c["slopes"]:
                s = s - st["slopes"].view(hkv, g, 1, 1) * d.abs()
            see = d >= 0
            if c["prefix"]:
                see = see | (j < st["prefix_host"][i])
            if c["window"]:
                see = see & (d < c["window"])
            if c["first"]:
                see = see & (j >= st["first_host"][i])
            s = s.masked_fill(~see, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
            l = p.sum(-1, keepdim=True)
            o = (p.view(hkv, g * (b - a), total) @ v).view(hkv, g, b - a, hd) / torch.where(l == 0, torch.ones_like(l), l)
            out[at + a:at + b] = o.permute(2, 0, 1, 3).reshape(b - a, n_head, hd).to(out.dtype)
        at += n
    return out


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return (_plain_plan if op == "plan" else _plain_store if op == "store" else _plain_attention)(state)


# ---- the definitions in 64 bits --------------------------------------------------

def _exact_plan(st):
    page, n_seq = st["case"]["page"], st["case"]["n_seq"]
    table = st["table"].cpu().numpy().copy()
    stack = st["free"][:int(st["n_free"])].cpu().tolist()
    cu, slot, pos = [0], [], []
    for i in range(n_seq):
        p, n = st["past_host"][i], st["new_host"][i]
        for col in range(-(-p // page), -(-(p + n) // page)):
            table[i, col] = stack.pop()
        ps = np.arange(p, p + n, dtype=np.int64)
        pos.append(ps)
        slot.append(table[i, ps // page].astype(np.int64) * page + ps % page)
        cu.append(cu[-1] + n)
    return (torch.from_numpy(table), torch.tensor(cu, dtype=torch.int32), torch.tensor(st["total_host"], dtype=torch.int32),
            torch.from_numpy(np.concatenate(slot)), torch.from_numpy(np.concatenate(pos).astype(np.int32)),
            torch.tensor([len(stack)], dtype=torch.int32))


def _exact_rope(x, pos, st):
    """x [n][heads][hd] f64, pairs as complex numbers turned by their angle's table entries."""
    hd = x.shape[-1]
    turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None]
    if SHAPES[st["case"]["shape"]][3]:
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
        return torch.cat((z.real, z.imag), -1)
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], hd // 2, 2).contiguous()) * turn
    return torch.view_as_real(z).reshape(x.shape)


def _exact_store(st):
    c = st["case"]
    page = c["page"]
    k, v = st["dk"].double(), st["dv"].double()
    if c["rope"]:
        k = _exact_rope(k, st["pos"].long(), st)
    slot = st["slot"]
    outs = []
    for x, codes, scale in ((k, st["k"], st["k_scale"]), (v, st["v"], st["v_scale"])):
        # the touched blocks as a dense [block][16][hkv][hd] batch of values and codes
        ids, inv = torch.unique(slot // BLOCK, return_inverse=True)
        n, (hkv, hd) = ids.numel(), x.shape[1:]
        dense = torch.zeros(n, BLOCK, hkv, hd, dtype=torch.float64, device=x.device)
        fresh = torch.zeros(n, BLOCK, dtype=torch.bool, device=x.device)
        dense[inv, slot % BLOCK] = x
        fresh[inv, slot % BLOCK] = True
        every = ids[:, None] * BLOCK + torch.arange(BLOCK, device=x.device)
        kept = codes[every // page, :, every % page].double()
        lead = fresh.int().argmax(1)                      # rows before the first new one are valid
        old = scale[ids * BLOCK // page, :, ids * BLOCK % page // BLOCK].double()
        old = torch.where((lead > 0)[:, None], old, torch.zeros_like(old))
        new = torch.maximum(old, dense.abs().amax((1, 3)) / 127)
        safe = torch.where(new > 0, new, torch.ones_like(new))
        q = torch.round(dense / safe[:, None, :, None])
        q = torch.where(fresh[:, :, None, None], q, torch.round(kept * (old / safe)[:, None, :, None]))
        val = q * new[:, None, :, None]
        at = torch.searchsorted(ids, st["back"] // BLOCK)
        outs.append(val[at, st["back"] % BLOCK])
    return tuple(outs)


def _exact_attention(st):
    c = st["case"]
    n_head, hkv, hd, _, _ = SHAPES[c["shape"]]
    g, page = n_head // hkv, c["page"]
    dev = st["q"].device
    out = torch.zeros(st["n_tok"], n_head, hd, dtype=torch.float64, device=dev)
    cu = [0]
    for n in st["new_host"]:
        cu.append(cu[-1] + n)
    for i in range(c["n_seq"]):
        n, total = st["new_host"][i], st["total_host"][i]
        if not n:
            continue
        row_pos = torch.arange(total - n, total, device=dev)
        q = st["q"][cu[i]:cu[i + 1]].double()
        if c["rope"]:
            q = _exact_rope(q, row_pos, st)
        j = torch.arange(total, device=dev)
        pg, off = st["table"][i][j // page].long(), j % page
        for h in range(n_head):
            kh = h // g
            key = st["k"][pg, kh, off].double() * st["k_scale"][pg, kh, off // BLOCK].double()[:, None]
            val = st["v"][pg, kh, off].double() * st["v_scale"][pg, kh, off // BLOCK].double()[:, None]
            step = max(1, (1 << 26) // total)
            for a in range(0, n, step):
                p = row_pos[a:a + step, None]
                z = torch.einsum("rd,jd->rj", q[a:a + step, h], key) * st["scale"]
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                if c["slopes"]:
                    z -= float(st["slopes"][h]) * (p - j).abs().double()
                hidden = j > p
                if c["prefix"]:
                    hidden &= j >= st["prefix_host"][i]
                if c["window"]:
                    hidden |= j <= p - c["window"]
                if c["first"]:
                    hidden |= j < st["first_host"][i]
                z[hidden] = -math.inf
                w = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
                out[cu[i] + a:cu[i] + a + w.shape[0], h] = torch.einsum("rj,jd->rd", torch.nan_to_num_(w), val)
    return out


def exact(case, seed):
    st = _inputs(case, seed)
    op = case["op"]
    return (_exact_plan if op == "plan" else _exact_store if op == "store" else _exact_attention)(st)
