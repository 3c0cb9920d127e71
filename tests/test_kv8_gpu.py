"""The paged 8-bit KV cache on the device (sicu_kv8_*) against plain numpy in
64 bits: block tables, the quantizing store, attention with its masks."""

from __future__ import annotations

import numpy as np
import pytest

from siphon_b200 import lib as L
from tests import kv8_ref as R
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu


def i32(a):
    return dev(np.asarray(a, np.int32))


def spread(n_seq, page, lens, rng, spare=3):
    """A table whose requests own shuffled pages, the pool size and the rest."""
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + spare
    order = rng.permutation(n_pages).astype(np.int32)
    table = np.zeros((n_seq, max(max(need), 1)), np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, n_pages, order[at:]


# ---- block tables and slot maps ------------------------------------------------------

@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n_seq,past_hi,new_hi,extra", [(1, 0, 1, 0), (1, 500, 1, 3), (7, 200, 40, 0), (64, 2000, 1, 5),
                                                       (1500, 300, 9, 1), (5000, 40, 2, 0), (3, 0, 5000, 2)])
def test_plan(sicu, page, n_seq, past_hi, new_hi, extra):
    import torch
    rng = np.random.default_rng(n_seq * 7 + page)
    past = rng.integers(0, past_hi + 1, n_seq)
    fresh = rng.integers(0, new_hi + 1, n_seq)
    need = [-(-int(p + f) // page) for p, f in zip(past, fresh)]
    held = [-(-int(p) // page) for p in past]
    table, n_pages, free = spread(n_seq, page, [h * page for h in held], rng, spare=sum(need) - sum(held) + 2)
    width = max(max(need), 1)
    wide = np.full((n_seq, width), -7, np.int32)
    wide[:, :table.shape[1]] = table[:, :width]
    w_table, w_cu, w_len, w_slot, w_pos, w_stack = R.plan(past, fresh, page, wide, free)
    stack = np.concatenate([free, np.zeros(n_pages - len(free), np.int32)])
    n_tok = int(fresh.sum())
    for alias in (False, True):        # outputs of their own, and in place of the inputs
        d_past, d_free, d_nf, d_table = i32(past), dev(stack), i32([len(free)]), dev(wide)
        d_len = d_past if alias else torch.full((n_seq,), -1, dtype=torch.int32, device="cuda")
        d_out = d_nf if alias else i32([-1])
        cu = torch.full((n_seq + 1,), -1, dtype=torch.int32, device="cuda")
        slot = torch.full((n_tok + extra,), -9, dtype=torch.int64, device="cuda")
        pos = torch.full((n_tok + extra,), -9, dtype=torch.int32, device="cuda")
        sicu.kv8_plan(d_past, i32(fresh), n_seq, page, d_table, width, d_free, n_pages, d_nf, d_out, n_tok + extra, cu,
                      d_len, slot, pos)
        assert (host(d_table) == w_table).all() and (host(cu) == w_cu).all() and (host(d_len) == w_len).all()
        assert (host(slot)[:n_tok] == w_slot).all() and (host(pos)[:n_tok] == w_pos).all()
        assert (host(slot)[n_tok:] == -1).all() and (host(pos)[n_tok:] == 0).all()
        assert host(d_out)[0] == len(w_stack) and (host(d_free) == stack).all()
    assert sicu.status() == 0


@pytest.mark.parametrize("why", ["pages", "tokens", "width", "negative", "stack"])
def test_plan_places_nothing_when_it_does_not_fit(sicu, why):
    import torch
    page, past, fresh, n_free, n_tok, width = 16, [5, 17, 0], [20, 3, 40], 9, 63, 4
    want = L.STATUS_BAD_PLAN
    if why == "pages":
        n_free, want = 3, L.STATUS_NO_PAGES       # 1 + 0 + 3 pages needed
    elif why == "tokens":
        n_tok = 62
    elif why == "width":
        width = 2
    elif why == "negative":
        fresh = [20, -3, 40]
    else:
        n_free = 31
    table = np.arange(3 * width, dtype=np.int32).reshape(3, width)
    d_table, cu = dev(table), torch.full((4,), -1, dtype=torch.int32, device="cuda")
    length, out = torch.full((3,), -1, dtype=torch.int32, device="cuda"), i32([-1])
    slot = torch.zeros(n_tok, dtype=torch.int64, device="cuda")
    pos = torch.full((n_tok,), 5, dtype=torch.int32, device="cuda")
    sicu.kv8_plan(i32(past), i32(fresh), 3, page, d_table, width, i32(np.arange(30)), 30, i32([n_free]), out, n_tok, cu,
                  length, slot, pos)
    assert sicu.status() == want
    assert (host(d_table) == table).all() and (host(cu) == 0).all() and (host(length) == past).all()
    assert (host(slot) == -1).all() and (host(pos) == 0).all() and host(out)[0] == n_free


def test_plan_leaves_out_tokens_of_pages_outside_the_pool(sicu):
    import torch
    # request 0 goes on in a held page, 1 takes the stack's top two, 2 the one below
    table = np.array([[-3, 0], [0, 0], [0, 0], [7, 0]], np.int32)
    stack = i32([0, 1, 2, 3, 12, 5, 10, 0, 0, 0])     # ids 0 .. 9; n_free 7: takes 10, 5, then 12
    cu, length = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    slot = torch.zeros(24, dtype=torch.int64, device="cuda")
    pos = torch.zeros(24, dtype=torch.int32, device="cuda")
    sicu.kv8_plan(i32([3, 0, 0, 2]), i32([1, 18, 2, 1]), 4, 16, dev(table), 2, stack, 10, i32([7]), i32([0]), 24, cu,
                  length, slot, pos)
    assert sicu.status() == L.STATUS_BAD_PLAN
    assert host(slot).tolist() == [-1] + [-1] * 16 + [80, 81] + [-1, -1] + [7 * 16 + 2] + [-1, -1]
    assert host(length).tolist() == [4, 18, 2, 3] and host(cu).tolist() == [0, 1, 19, 21, 22]


def test_release_and_reuse(sicu):
    page, width = 16, 4
    table = np.arange(20, dtype=np.int32).reshape(5, width)
    lens = np.array([33, 0, 64, 1, 16], np.int32)
    stack = np.concatenate([[90, 91], np.zeros(98)]).astype(np.int32)
    d_len, d_stack, d_n = dev(lens), dev(stack), i32([2])
    sicu.kv8_release(i32([1, 1, 0, 7, -1]), d_len, 5, page, dev(table), width, d_stack, 100, d_n)
    assert host(d_len).tolist() == [0, 0, 64, 0, 0]
    assert host(d_n)[0] == 2 + 3 + 0 + 1 + 1
    assert host(d_stack)[:7].tolist() == [90, 91, 0, 1, 2, 12, 16]
    assert sicu.status() == 0
    # lengths past the table, or a stack that would outgrow the pool: nothing changes
    d_len = dev(np.array([33, 0, 65, 1, 16], np.int32))
    sicu.kv8_release(i32([0, 0, 1, 1, 0]), d_len, 5, page, dev(table), width, d_stack, 100, d_n)
    assert sicu.status() == L.STATUS_BAD_PLAN and host(d_n)[0] == 7 and host(d_len)[3] == 1
    sicu.kv8_release(i32([0, 0, 0, 1, 0]), d_len, 5, page, dev(table), width, d_stack, 7, d_n)
    assert sicu.status() == L.STATUS_BAD_PLAN and host(d_n)[0] == 7


# ---- store and load ---------------------------------------------------------------------

def make_cache(n_pages, hkv, page, hd, rng):
    """Caches full of stale codes and scales, on the host and the device."""
    k, v = R.Cache(n_pages, hkv, page, hd), R.Cache(n_pages, hkv, page, hd)
    for c in (k, v):
        c.codes[:] = rng.integers(-127, 128, c.codes.shape)
        c.scale[:] = rng.uniform(0.01, 0.05, c.scale.shape)
    bufs = [dev(k.codes), dev(v.codes), dev(k.scale), dev(v.scale)]
    return k, v, bufs, L.kv8_cache(*bufs, n_pages, page, hkv, hd)


@pytest.mark.parametrize("hd,hkv,page", [(64, 4, 16), (96, 3, 32), (128, 8, 64), (256, 2, 128)])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("neox,n_rot", [(False, None), (True, None), (True, 32), (False, 0)])
def test_store_matches_bit_for_bit(sicu, hd, hkv, page, f16, neox, n_rot):
    """Codes and scales equal the stated f32 arithmetic exactly: prompts, rows
    appended mid-block over several steps with growing magnitudes (so blocks
    are requantized), skipped tokens, strided rows."""
    import torch
    rng = np.random.default_rng(hd + page + f16)
    n_rot = hd if n_rot is None else n_rot
    lens = [0, 5, 16, 61, 3]
    steps = [[37, 1, 16, 70, 0], [1, 1, 1, 1, 1], [1, 9, 1, 0, 13], [2, 1, 31, 1, 1]]
    total = [a + sum(s[i] for s in steps) for i, a in enumerate(lens)]
    table, n_pages, _ = spread(5, page, total, rng)
    k, v, bufs, cache = make_cache(n_pages, hkv, page, hd, rng)
    cos, sin = R.rope_tables(max(total), max(n_rot, 2))
    rope = L.rope(dev(cos), dev(sin), max(total), n_rot, neox) if n_rot else None
    keep = (rope, cos, sin)
    t_cos, t_sin = dev(cos), dev(sin)
    if n_rot:
        rope = L.rope(t_cos, t_sin, max(total), n_rot, neox)
    dt = np.float16 if f16 else np.float32
    past = list(lens)
    for step, fresh in enumerate(steps):
        slot, pos = [], []
        for i, f in enumerate(fresh):
            for p in range(past[i], past[i] + f):
                slot.append(int(table[i, p // page]) * page + p % page)
                pos.append(p)
            past[i] += f
        n = len(slot)
        slot, pos = np.array(slot, np.int64), np.array(pos, np.int32)
        if step == 1:
            slot[2] = -1
        pad = 32                                            # q, k and v rows of one buffer
        x = (rng.standard_normal((n, 2 * hkv * hd + pad)) * (1 + 2 * step)).astype(dt)
        x[:, 3] *= 20
        kx = x[:, :hkv * hd].reshape(n, hkv, hd).astype(np.float32)
        vx = x[:, hkv * hd:2 * hkv * hd].reshape(n, hkv, hd).astype(np.float32)
        if n_rot:
            kx = R.rotate(kx, pos, cos, sin, n_rot, neox)
        k.store(kx, slot)
        v.store(vx, slot)
        d = dev(x)
        sicu.kv8_store(cache, L.T_F16 if f16 else L.T_F32, d, d.data_ptr() + hkv * hd * x.itemsize, dev(slot), n,
                       pos=dev(pos), rope=rope, k_stride=x.shape[1], v_stride=x.shape[1])
        for got, want in zip(bufs, (k.codes, v.codes, k.scale, v.scale)):
            assert (host(got) == want).all(), f"step {step}"
    del keep
    # the stored rows as values
    rows = np.array([int(table[i, p // page]) * page + p % page for i in range(5) for p in range(past[i])] + [-1], np.int64)
    out = [torch.full((len(rows), hkv, hd), 9.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
           for _ in range(2)]
    sicu.kv8_load(cache, L.T_F16 if f16 else L.T_F32, dev(rows), len(rows), *out)
    for got, c in zip(out, (k, v)):
        want = c.codes[rows // page, :, rows % page].astype(np.float32) * \
            c.scale[rows // page, :, rows % page // R.BLOCK][..., None]
        want[-1] = 0
        assert (host(got) == want.astype(dt)).all()
    assert sicu.status() == 0


def test_store_of_zeros_tiny_and_nonfinite_values(sicu):
    rng = np.random.default_rng(5)
    hkv, hd, page = 2, 64, 16
    k, v, bufs, cache = make_cache(4, hkv, page, hd, rng)
    x = rng.standard_normal((20, hkv, hd)).astype(np.float32)
    x[:16, 0] = 0.0                                  # a whole block of zeros
    x[:16, 1] *= np.float32(2.0 ** -120)             # too small for a scale
    y = x.copy()
    y[3, 0, 5], y[17, 1, 7], y[18, 1, 8], y[19, 0, 0] = np.nan, np.inf, -np.inf, np.nan
    slot = np.arange(16, 36, dtype=np.int64)
    k.store(x, slot)
    v.store(y, slot)
    sicu.kv8_store(cache, L.T_F32, dev(x), dev(y), dev(slot), 20)
    for got, want in zip(bufs, (k.codes, v.codes, k.scale, v.scale)):
        assert (host(got) == want).all()
    assert sicu.status() == L.STATUS_NONFINITE
    assert k.scale[1, 0, 0] == 0 and k.scale[1, 1, 0] == 0 and not k.codes[1].any()
    assert v.codes[2, 1, 1, 7] == 127 and v.codes[2, 1, 2, 8] == -127 and v.codes[2, 0, 3, 0] == 0


def test_slots_outside_the_pool_are_left_out(sicu):
    import torch
    rng = np.random.default_rng(6)
    k, v, bufs, cache = make_cache(3, 1, 16, 64, rng)
    x = rng.standard_normal((3, 1, 64)).astype(np.float32)
    slot = np.array([48, 5000000000, 0], np.int64)      # the second and the first past the 3 pages
    k.store(x[2:], slot[2:])
    v.store(x[2:], slot[2:])
    sicu.kv8_store(cache, L.T_F32, dev(x), dev(x), dev(slot), 3)
    for got, want in zip(bufs, (k.codes, v.codes, k.scale, v.scale)):
        assert (host(got) == want).all()
    assert sicu.status() == L.STATUS_BAD_PLAN
    out = torch.ones(3, 64, device="cuda")
    sicu.kv8_load(cache, L.T_F32, dev(slot), 3, out, torch.ones_like(out))
    assert (host(out)[:2] == 0).all() and host(out)[2].any()
    assert sicu.status() == L.STATUS_BAD_PLAN


# ---- attention ------------------------------------------------------------------------------

def attend(sicu, n_head, hkv, hd, page, past, fresh, f16=False, cap=0.0, slopes=False, window=0, prefix=None, first=None,
           neox=False, n_rot=None, seed=0, qmul=2.0, stride_pad=0, stream=None, edit=None):
    """Runs one call and checks it: every output within the bound derived here."""
    import torch
    rng = np.random.default_rng(seed)
    lens = [p + f for p, f in zip(past, fresh)]
    n_rot = hd if n_rot is None else n_rot
    table, n_pages, _ = spread(len(lens), page, lens, rng)
    k, v, bufs, cache = make_cache(n_pages, hkv, page, hd, rng)
    if edit:
        edit(k, v, bufs, table)
    cu = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
    n = int(cu[-1])
    dt = np.float16 if f16 else np.float32
    wide = rng.standard_normal((max(n, 1), n_head * hd + stride_pad)) * qmul
    wide = wide.astype(dt)
    q = wide[:n, :n_head * hd].reshape(n, n_head, hd)
    rows = max(max(lens), 1)
    cos, sin = R.rope_tables(rows, max(n_rot, 2))
    d_cos, d_sin = dev(cos), dev(sin)
    rope = L.rope(d_cos, d_sin, rows, n_rot, neox) if n_rot else None
    pos = np.concatenate([np.arange(p, p + f) for p, f in zip(past, fresh)]).astype(np.int64)
    q64 = q.astype(np.float64)
    if n_rot:
        q64 = R.rotate(q64, pos, cos.astype(np.float64), sin.astype(np.float64), n_rot, neox)
    sl = 2.0 ** (-8.0 * (np.arange(n_head) + 1) / n_head) if slopes else None
    scale = float(np.float32(1 / np.sqrt(hd)))
    want, top = R.attention(q64, k, v, table, lens, cu, scale, cap, sl, window, prefix, first)
    d_q, d_table, d_len, d_cu = dev(wide), dev(table), i32(lens), dev(cu)
    d_sl = dev(sl.astype(np.float32)) if slopes else None
    d_pre = i32(prefix) if prefix is not None else None
    d_first = i32(first) if first is not None else None
    out = torch.full((max(n, 1), n_head * hd + stride_pad), 7.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    at = L.kv8_attn(L.T_F16 if f16 else L.T_F32, n_head, n, d_table, table.shape[1], d_len, d_cu, len(lens), max(fresh),
                    max(lens), scale, cap=cap, slopes=d_sl, window=window, prefix=d_pre, first=d_first, rope=rope,
                    q_stride=n_head * hd + stride_pad, out_stride=n_head * hd + stride_pad)
    ws = torch.full((max(sicu.kv8_attention_ws(cache, at), 16),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    sicu.kv8_attention(cache, at, d_q, out, ws, stream=stream)
    got = host(out).astype(np.float64)
    assert (got[n:] == 7).all() and (got[:n, n_head * hd:] == 7).all(), "written outside the rows"
    got = got[:n, :n_head * hd].reshape(n, n_head, hd)
    assert sicu.status() == 0
    # Scores: f32 sums of hd exact products of 22-bit parts of q, RoPE's and the
    # scale's roundings: within (hd / 4 + 16) 2^-24 of the largest |score|'s size
    # times the cancellation sum|q k| / |q . k| ~ sqrt(hd); the cap's own error
    # 2^-20 cap; the slope term's 2^-23 of slope * distance. A score error d
    # moves weights by d relatively, the output by 2 d max|v|; the exponential
    # and the sums add 2^-20. f16 callers: weights rounded to 2^-11 and the
    # output to 2^-11 of itself.
    size = (top + 1) * np.sqrt(hd)
    d = size * (hd / 4 + 16) * 2.0 ** -24 + cap * 2.0 ** -20 + (max(lens) * 2.0 ** -23 if slopes else 0) + 2.0 ** -20
    vmax = float(np.abs(v.codes.astype(np.float64)).max() * np.nanmax(v.scale))
    tol = vmax * 2 * d + (vmax * 2.0 ** -10 if f16 else 0)
    err = np.abs(got - want)
    assert not np.isnan(got).any() and err.max() <= tol, f"max error {err.max():.3g} > {tol:.3g}"
    return got, want


LAYOUTS = [(8, 2, 64), (32, 4, 64), (4, 4, 96), (32, 8, 128), (40, 8, 128), (16, 1, 128), (8, 4, 256), (48, 2, 64)]


@pytest.mark.parametrize("n_head,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("f16", [False, True])
def test_attention_single_tokens(sicu, n_head, hkv, hd, f16):
    """One new token each: lengths of one, around block, page and split ends."""
    past = [0, 1, 14, 15, 16, 31, 63, 64, 65, 255, 256, 300, 700]
    attend(sicu, n_head, hkv, hd, 16, past, [1] * len(past), f16=f16, neox=f16, seed=hd + n_head)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_pages_and_idle_requests(sicu, page):
    attend(sicu, 8, 2, 64, page, [0, 100, 17, 0, 333], [1, 0, 1, 0, 1], seed=page)
    attend(sicu, 8, 2, 64, page, [0, 100, 17, 0, 333], [3, 0, 40, 1, 2], seed=page + 1, stride_pad=16)


@pytest.mark.parametrize("n_head,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("f16", [False, True])
def test_attention_prompts(sicu, n_head, hkv, hd, f16):
    """Several new tokens: first prompts, continued ones, ragged ends."""
    attend(sicu, n_head, hkv, hd, 32, [0, 5, 130, 31], [70, 33, 2, 1], f16=f16, neox=True, seed=hd * 3 + n_head)


@pytest.mark.parametrize("fresh", [[1, 1, 1, 1], [50, 1, 20, 90]])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("mask", ["cap", "slopes", "window", "prefix", "first", "all"])
def test_attention_masks_and_scores(sicu, fresh, f16, mask):
    past = [0, 40, 200, 7]
    lens = [p + f for p, f in zip(past, fresh)]
    kw = {}
    if mask in ("cap", "all"):
        kw["cap"] = 5.0
    if mask in ("slopes", "all"):
        kw["slopes"] = True
    if mask in ("window", "all"):
        kw["window"] = 19
    if mask in ("prefix", "all"):
        kw["prefix"] = [lens[0], 0, 130, lens[3] // 2]
    if mask in ("first", "all"):
        # some rows, and the whole of the third request, see nothing
        kw["first"] = [0, 41, lens[2], 3]
    for nh, hkv, hd in ((8, 2, 64), (10, 2, 128)):
        got, want = attend(sicu, nh, hkv, hd, 16, past, fresh, f16=f16, seed=len(mask), **kw)
        if "first" in kw and "prefix" not in kw:
            c = fresh[0] + fresh[1]
            assert (got[c:c + fresh[2]] == 0).all()


@pytest.mark.parametrize("window", [1, 15, 16, 17, 10 ** 9])
def test_attention_windows(sicu, window):
    attend(sicu, 8, 2, 64, 16, [0, 90, 33], [1, 1, 1], window=window, seed=window % 97)
    attend(sicu, 8, 2, 64, 16, [0, 90, 33], [40, 3, 17], window=window, seed=window % 97)


@pytest.mark.parametrize("n_rot,neox", [(0, False), (32, False), (32, True)])
def test_attention_partial_rotation(sicu, n_rot, neox):
    attend(sicu, 8, 2, 64, 16, [0, 70], [1, 1], n_rot=n_rot, neox=neox)
    attend(sicu, 8, 2, 64, 16, [0, 70], [9, 30], n_rot=n_rot, neox=neox)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("fresh", [1, 80])
def test_attention_long_and_extreme_scales(sicu, f16, fresh):
    """Thousands of keys over many splits, V scales far apart and of zero, a
    very large score on one key."""
    def edit(k, v, bufs, table):
        v.scale[::3] *= 1e-6
        v.scale[1::3] = 0.0
        v.codes[1::3] = 0
        k.scale[2] *= 30
        for b, a in zip(bufs, (k.codes, v.codes, k.scale, v.scale)):
            b.copy_(dev(a))
    attend(sicu, 4, 1, 64, 64, [5000], [fresh], f16=f16, edit=edit, seed=9)
    attend(sicu, 8, 2, 128, 16, [3000], [fresh], f16=f16, seed=10)


def test_attention_reads_nothing_outside_a_request(sicu):
    """Stale codes and scales in the rows past a length and in pages of nobody
    do not reach the result, whatever bits they hold."""
    def edit(k, v, bufs, table):
        used = np.zeros(k.codes.shape[0], bool)
        used[table[0, :3]] = True                    # 40 tokens of 16: pages 0..2 of the table
        for c in (k, v):
            c.scale[~used] = np.nan
            c.codes[table[0, 2], :, 8:] = -128
        for b, a in zip(bufs, (k.codes, v.codes, k.scale, v.scale)):
            b.copy_(dev(a))
    attend(sicu, 8, 2, 64, 16, [39], [1], edit=edit)
    attend(sicu, 8, 2, 64, 16, [10], [30], edit=edit)


def test_attention_evicted_pages_are_not_read(sicu):
    """Pages wholly before first[i] may already belong to someone else."""
    def edit(k, v, bufs, table):
        gone = table[0, :4].copy()
        for c in (k, v):
            c.scale[gone] = np.inf
        for b, a in zip(bufs, (k.codes, v.codes, k.scale, v.scale)):
            b.copy_(dev(a))
        table[0, :4] = 0
        for c in (k, v):
            c.scale[gone] = 0.01                     # for the plain form, which masks after reading
    attend(sicu, 8, 2, 64, 16, [200], [1], first=[70], edit=edit)
    attend(sicu, 8, 2, 64, 16, [200], [20], first=[70], edit=edit)


def test_attention_nan_query_gives_nan(sicu):
    import torch
    rng = np.random.default_rng(3)
    for n in (1, 70):
        table, n_pages, _ = spread(1, 16, [n], rng)
        k, v, bufs, cache = make_cache(n_pages, 2, 16, 64, rng)
        q = rng.standard_normal((n, 8, 64)).astype(np.float32)
        q[0, 3, 7] = np.nan
        out = torch.zeros(n, 8, 64, device="cuda")
        d_table, d_len, d_cu = dev(table), i32([n]), i32([0, n])
        at = L.kv8_attn(L.T_F32, 8, n, d_table, table.shape[1], d_len, d_cu, 1, n, n, 0.125)
        ws = torch.empty(max(sicu.kv8_attention_ws(cache, at), 16), dtype=torch.uint8, device="cuda")
        sicu.kv8_attention(cache, at, dev(q), out, ws)
        got = host(out)
        assert np.isnan(got[0, 3]).all()
        ok = np.ones((n, 8), bool)
        ok[0, 3] = False
        assert np.isfinite(got[ok]).all()


@pytest.mark.parametrize("what", ["len", "cu", "new", "page"])
def test_attention_refuses_device_numbers_out_of_range(sicu, what):
    """A request whose numbers pass the host's bounds is left out, with the
    status bit; a page id outside the pool reads page 0."""
    import torch
    rng = np.random.default_rng(4)
    for fresh in ([1, 1], [40, 40]):
        lens = [60, 50]
        table, n_pages, _ = spread(2, 16, lens, rng)
        k, v, bufs, cache = make_cache(n_pages, 2, 16, 64, rng)
        cu = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
        n, max_new = int(cu[-1]), max(fresh)
        if what == "len":
            lens = [60, 4000]
        elif what == "cu":
            cu[2] = n + 1
        elif what == "new":
            max_new -= 1 if max_new > 1 else 0
            if max_new == 1:
                lens = [60, 0]
        else:
            table[1, 0] = n_pages
        q = rng.standard_normal((n, 8, 64)).astype(np.float32)
        out = torch.full((n, 8, 64), 7.0, device="cuda")
        d_table, d_len, d_cu = dev(table), i32(lens), dev(cu)
        at = L.kv8_attn(L.T_F32, 8, n, d_table, table.shape[1], d_len, d_cu, 2, max_new, 60, 0.125)
        ws = torch.empty(max(sicu.kv8_attention_ws(cache, at), 16), dtype=torch.uint8, device="cuda")
        sicu.kv8_attention(cache, at, dev(q), out, ws)
        got = host(out)
        assert sicu.status() == L.STATUS_BAD_PLAN
        if what == "page":
            assert np.isfinite(got).all() and (got != 7).all()
        else:
            assert (got[cu[1]:] == 7).all()


def test_calls_repeat_bit_for_bit_on_another_stream_and_in_a_graph(sicu):
    import torch
    rng = np.random.default_rng(12)
    past, fresh, page = [900, 20, 0, 450], [1, 60, 3, 1], 32
    lens = [p + f for p, f in zip(past, fresh)]
    table, n_pages, _ = spread(4, page, lens, rng)
    k, v, bufs, cache = make_cache(n_pages, 2, page, 128, rng)
    n = sum(fresh)
    q, kx, vx = (dev(rng.standard_normal((n, h * 128)).astype(np.float32)) for h in (8, 2, 2))
    slot = np.array([int(table[i, p // page]) * page + p % page for i in range(4) for p in range(past[i], lens[i])], np.int64)
    d_slot, d_table, d_len = dev(slot), dev(table), i32(lens)
    d_cu = i32(np.concatenate([[0], np.cumsum(fresh)]))
    at = L.kv8_attn(L.T_F32, 8, n, d_table, table.shape[1], d_len, d_cu, 4, max(fresh), max(lens), 0.088)
    ws = torch.empty(max(sicu.kv8_attention_ws(cache, at), 16), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()

    def step(h):
        sicu.kv8_store(cache, L.T_F32, kx, vx, d_slot, n, stream=h)
        sicu.kv8_attention(cache, at, q, out, ws, stream=h)

    step(side.cuda_stream)
    side.synchronize()
    first = host(out).copy()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for _ in range(3):
        out.fill_(3.0)
        graph.replay()
        assert (host(out) == first).all()
    assert sicu.status() == 0


def test_attention_prompt_f32_precision_over_many_keys(sicu):
    """A chunk far into a long context: f32 results stay as close to 64 bits as
    sums in f32 do (the bound of `attend` without its slack for the scores:
    here every score is small, so the sums over 6000 keys are what can err)."""
    got, want = attend(sicu, 4, 1, 128, 64, [6000], [40], qmul=0.02, seed=21)
    # 6000 weights near 1 / 6000 of values of unit size: the result is their
    # mean, some 1 / sqrt(6000) of them; an f32 sum errs by 2^-24 sqrt(6000) of
    # its terms' size, the weights by 2^-22 each
    err = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert err < 2.0 ** -18


def test_pool_past_32_bits(sicu):
    """Pages whose codes begin past 2^32 elements: store, load and both
    attention kernels reach them (a pool of 5.2 GB for K alone)."""
    import torch
    hkv, hd, page, n_pages = 8, 128, 128, 40000
    bufs = [torch.zeros(n_pages, hkv, page, hd, dtype=torch.int8, device="cuda") for _ in range(2)] + \
           [torch.zeros(n_pages, hkv, page // 16, device="cuda") for _ in range(2)]
    cache = L.kv8_cache(*bufs, n_pages, page, hkv, hd)
    rng = np.random.default_rng(8)
    pages = [39999, 12, 38001]
    n = 300
    slot = np.array([pages[p // page] * page + p % page for p in range(n)], np.int64)
    x = rng.standard_normal((2, n, hkv, hd)).astype(np.float32)
    small = [R.Cache(3, hkv, page, hd) for _ in range(2)]            # the same rows in pages 0, 1, 2
    for c, v in zip(small, x):
        c.store(v, np.arange(n, dtype=np.int64))
    sicu.kv8_store(cache, L.T_F32, dev(x[0]), dev(x[1]), dev(slot), n)
    out = [torch.empty(n, hkv, hd, device="cuda") for _ in range(2)]
    sicu.kv8_load(cache, L.T_F32, dev(slot), n, *out)
    for got, c in zip(out, small):
        assert np.allclose(host(got), c.load(np.arange(n)), rtol=2.0 ** -22, atol=0)
    for new in (1, 60):
        q = rng.standard_normal((new, 16, hd)).astype(np.float32)
        want, _ = R.attention(q.astype(np.float64), *small, np.array([[0, 1, 2]], np.int32), [n], [0, new], 0.088)
        o = torch.empty(new, 16, hd, device="cuda")
        d_table, d_len, d_cu = i32([pages]), i32([n]), i32([0, new])
        at = L.kv8_attn(L.T_F32, 16, new, d_table, 3, d_len, d_cu, 1, new, n, 0.088)
        ws = torch.empty(max(sicu.kv8_attention_ws(cache, at), 16), dtype=torch.uint8, device="cuda")
        sicu.kv8_attention(cache, at, dev(q), o, ws)
        # scores of a few units in f32, values of 4 at most
        assert np.abs(host(o) - want).max() < 4 * 2.0 ** -17
    assert sicu.status() == 0


def test_positions_past_the_rope_tables_are_reported(sicu):
    import torch
    rng = np.random.default_rng(9)
    k, v, bufs, cache = make_cache(8, 2, 16, 64, rng)
    cos, sin = R.rope_tables(40, 64)
    d_cos, d_sin = dev(cos), dev(sin)
    rope = L.rope(d_cos, d_sin, 40, 64)
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    sicu.kv8_store(cache, L.T_F32, dev(x), dev(x), dev(np.arange(3, dtype=np.int64)), 3, pos=i32([39, 40, -1]), rope=rope)
    assert sicu.status() == L.STATUS_BAD_PLAN
    for new in (1, 50):
        q = rng.standard_normal((new, 8, 64)).astype(np.float32)
        out = torch.zeros(new, 8, 64, device="cuda")
        d_table, d_len, d_cu = i32([np.arange(8)]), i32([60]), i32([0, new])
        at = L.kv8_attn(L.T_F32, 8, new, d_table, 8, d_len, d_cu, 1, new, 60, 0.125, rope=rope)
        ws = torch.empty(max(sicu.kv8_attention_ws(cache, at), 16), dtype=torch.uint8, device="cuda")
        sicu.kv8_attention(cache, at, dev(q), out, ws)
        assert np.isfinite(host(out)).all()
        assert sicu.status() == L.STATUS_BAD_PLAN


@pytest.mark.parametrize("n_head,hkv,hd", [(8, 2, 64), (10, 2, 128)])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("mask", ["none", "cap", "steep cap", "slopes", "window", "prefix", "first", "all"])
def test_attention_masks_over_many_rows(sicu, n_head, hkv, hd, f16, mask):
    """Requests of several hundred rows (query heads x tokens), more than one
    tile of the tensor-memory kernel, next to short ones: full and partly
    filled tiles, spans that begin inside a block, rows and whole requests that
    see nothing, scores on both sides of half the cap."""
    past, fresh = [0, 40, 300, 7], [150, 1, 70, 133]
    lens = [p + f for p, f in zip(past, fresh)]
    kw = {"cap": {"cap": 200.0}, "steep cap": {"cap": 3.0}, "slopes": {"slopes": True}, "window": {"window": 37},
          "prefix": {"prefix": [lens[0], 0, 320, lens[3] // 2]}, "first": {"first": [100, 41, lens[2], 3]}, "none": {},
          "all": {"cap": 20.0, "slopes": True, "window": 61, "prefix": [20, 0, 340, 0], "first": [100, 0, 333, 140]}}[mask]
    got, want = attend(sicu, n_head, hkv, hd, 16, past, fresh, f16=f16, neox=f16, seed=3, **kw)
    if mask == "first":
        assert (got[:100] == 0).all() and (got[151:221] == 0).all() and got[100].any()
