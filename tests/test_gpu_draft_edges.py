"""Edges of the drafted-token operators on the GPU: counts and scales at the ends of what they may be, caches that hold rows of
zeros, what a caller may change between two calls."""
import numpy as np
import pytest
import torch

import draftref as ref
from test_gpu_draft import BF16, DEV, F16, F32, assert_within, gen, half_step, held_rows, i64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("none", [0, -1, -64, -(1 << 32) + 5, -(1 << 62)])
def test_keep_of_no_rows_leaves_the_cache(store, none):
    """A count of zero or less keeps nothing: codes and scales of every layer are as they were, the other sequences' rows move.
    The path's storage goes on behind its rows with numbers that are slots of the cache, so a read behind a row would show."""
    from sparse_transformers_b200 import KVCache

    L, B, kv, rows, hd = 2, 3, 2, 400, 32
    cache = KVCache(B, kv, rows, hd, dtype=F16, store=store, layers=L, device=DEV)
    g = gen(1)
    for i in range(L):
        x = torch.randn(B, rows, kv, hd, generator=g, device=DEV).to(F16)
        cache.layer(i).append(x, -2 * x, torch.zeros(B, dtype=torch.long, device=DEV))
    held = [t for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale) if t is not None]
    was = [t.clone() for t in held]
    block = torch.arange(B * 300, device=DEV).view(B, 300) % 90 + 7
    start, counts = i64(3, 10, 20), i64(none, 4, none)
    cache.keep(start, block[:, :64], counts)
    for now, old in zip(held, was):
        want = old.clone()
        for i in range(4):
            want[:, 1, :, 10 + i] = old[:, 1, :, 10 + int(block[1, i])]
        assert torch.equal(now, want)


def weight_slack(q, layer, length, counts, masks):
    """Elementwise bound for o = sum w_j v_j, relative to sum w_j |v_j| and not to the largest value of the cache.  A weight's relative
    error is at most twice its score's (its own and the sum's; a score's sum of hd products as in draftref.attention_slack) + half a
    step where it is held in 16 bits + 2^-16 for scores in powers of two of magnitude up to 64 in fp32 (2^-18 each for the product, the
    scale's logarithm, and both again in the sum).  In fp16 a weight times its row's scale (1 for 16-bit caches, 2^-40 for a row of
    zeros) is held as P with the largest such product at 2^7 at least: smaller than 2^-21 of it, P is a subnormal number and off
    by 2^-25, that is by 2^-32 of the largest product, times the row's code."""
    k, v = held_rows(layer)
    n = layer.k.shape[2]
    rel = ref.attention_slack(q, k, v, q.dtype) / float(v.abs().amax()) + 2.0 ** -16
    sum_abs = ref.attention(q, k, v.abs(), length, counts, masks, n)
    slack = rel * sum_abs
    if q.dtype == F16:
        s = torch.ones(layer.v.shape[:3], device=DEV).double() if layer.v_scale is None else layer.v_scale.double()
        one = torch.eye(n, dtype=torch.float64, device=DEV).expand(*k.shape[:2], n, n)
        wide = lambda t: torch.nn.functional.pad(t, (0, n - t.shape[-1]))  # as many values a head as there are slots
        w = ref.attention(wide(q), wide(k), one, length, counts, masks, n, q.shape[-1] ** -0.5)  # [B,T,heads,n]
        G = q.shape[2] // k.shape[1]
        most = (w * torch.where(s > 0, s, 2.0 ** -40).repeat_interleave(G, 1)[:, None]).amax(-1)
        codes = (layer.v.float().double().abs() * (s > 0)[..., None]).sum(2).repeat_interleave(G, 1)  # [B,heads,hd]
        slack = slack + 2.0 ** -32 * most[..., None] * codes[:, None]
    return slack


def zero_row_case(dtype, store, hd, T, amp, lead, n=300, zero=(5, 70, 131, 250), heads=4, kv=2, seed=0):
    """A cache whose values are of size amp, but for rows of zeros whose keys every query likes by `lead` more than the others."""
    from sparse_transformers_b200 import KVCache

    g = gen(seed)
    base = torch.randn(hd, generator=g, device=DEV)
    base *= hd ** 0.5 / base.norm()
    q = (base + 0.3 * torch.randn(2, T, heads, hd, generator=g, device=DEV)).to(dtype)
    rows = n + T
    k = 0.5 * torch.randn(2, rows, kv, hd, generator=g, device=DEV)
    v = amp * torch.randn(2, rows, kv, hd, generator=g, device=DEV)
    k[:, list(zero)] = base * lead / hd ** 0.5
    v[:, list(zero)] = 0
    layer = KVCache(2, kv, rows, hd, dtype=dtype, store=store, device=DEV).layer(0)
    layer.append(k.to(dtype), v.to(dtype), i64(0, 0))
    return layer, q, i64(n, n - 65)


@pytest.mark.parametrize("dtype,store", [(F16, "int8"), (F16, "e4m3"), (BF16, "int8"), (BF16, "e4m3"), (F32, "int8"), (F16, "same")])
@pytest.mark.parametrize("hd,T", [(64, 3), (128, 3), (128, 40), (256, 1), (256, 40)])
@pytest.mark.parametrize("amp", [1.0, 0.02, 0.002])
@pytest.mark.parametrize("lead", [0.0, 8.0, 12.0])
def test_value_rows_of_zeros_take_no_bits_from_the_others(dtype, store, hd, T, amp, lead):
    """A row of zeros (never written, padding, or flushed) adds to the soft-max's sum and to nothing else, whatever the other
    rows' scales are."""
    from sparse_transformers_b200 import tree_attention

    layer, q, length = zero_row_case(dtype, store, hd, T, amp, lead, seed=hd + T)
    k, v = held_rows(layer)
    want = ref.attention(q, k, v, length, None, None, layer.k.shape[2])
    assert_within(tree_attention(q, layer, length), want, half_step(want, dtype) + weight_slack(q, layer, length, None, None))


@pytest.mark.parametrize("dtype,store", [(F16, "int8"), (F16, "e4m3"), (BF16, "int8")])
@pytest.mark.parametrize("T", [3, 40])
def test_value_rows_of_very_different_sizes(dtype, store, T):
    """Rows from 2^-14 to 1, rows of zeros first, last and a whole tile of them; a cache of nothing but zeros gives zeros."""
    from sparse_transformers_b200 import tree_attention

    layer, q, length = zero_row_case(dtype, store, 128, T, 1.0, 6.0, zero=tuple(range(64)) + (299,), seed=T)
    g = gen(T + 1)
    size = 2.0 ** (-14 * torch.rand(2, 2, layer.k.shape[2], generator=g, device=DEV))
    layer.v_scale.mul_(size)
    k, v = held_rows(layer)
    want = ref.attention(q, k, v, length, None, None, layer.k.shape[2])
    assert_within(tree_attention(q, layer, length), want, half_step(want, dtype) + weight_slack(q, layer, length, None, None))
    layer.v.view(torch.uint8).zero_()
    layer.v_scale.zero_()
    assert bool((tree_attention(q, layer, length) == 0).all())


@pytest.mark.parametrize("mode", ["greedy", "tree", "chain"])
def test_verify_counts_far_from_the_nodes(mode):
    """A count is a 64-bit number: far below zero nothing is in use, far above all nodes are."""
    from sparse_transformers_b200 import verify_draft

    V, T = 40, 6
    counts = i64(-1, 0, -(1 << 32) + 3, -(1 << 63), T, T + 1, (1 << 32) + 1, (1 << 63) - 1)
    B = counts.numel()
    g = gen(4)
    p = torch.softmax(torch.randn(1, T, V, generator=g, device=DEV), -1).expand(B, T, V).contiguous()
    x, u = torch.randint(0, V, (1, T), generator=g, device=DEV).repeat(B, 1), torch.rand(1, T, generator=g, device=DEV).repeat(B, 1)
    if mode == "greedy":
        path, count, nxt = verify_draft(x, x.roll(-1, 1), counts=counts)
    elif mode == "tree":
        path, count, nxt = verify_draft(x, p, uniform=u, parents=torch.arange(-1, T - 1, device=DEV).repeat(B, 1), counts=counts)
    else:
        path, count, nxt = verify_draft(x, p, uniform=u, draft=p[:, 1:].contiguous(), counts=counts)
    assert bool((path[:4] == -1).all()) and count[:4].tolist() == [0] * 4 and nxt[:4].tolist() == [-1] * 4
    for b in range(5, B):
        assert torch.equal(path[b], path[4]) and count[b] == count[4] and nxt[b] == nxt[4]
    assert int(count[4]) >= 1 and int(nxt[4]) >= 0


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "int8"), (F16, "e4m3")])
@pytest.mark.parametrize("hd,T", [(64, 3), (128, 3), (128, 40), (256, 20)])
@pytest.mark.parametrize("copies", [0, 1, 4])
def test_expired_waits_are_reported(monkeypatch, dtype, store, hd, T, copies):
    """Thread blocks that do not request their keys wait for them until the limit: the call ends, what is on its way is drained, the rows
    are NaN, in units that several blocks share too, and the status says so, once."""
    from sparse_transformers_b200 import attention_timed_out, tree_attention
    from test_gpu_draft import attn_case

    layer, q, length, _, _ = attn_case(dtype, store, hd, 4, 2, T, [7000, 0, 30000], seed=hd)
    want = tree_attention(q, layer, length)
    assert not attention_timed_out()
    monkeypatch.setenv("STX_TREE_COPIES", str(copies))
    got = tree_attention(q, layer, length)
    assert attention_timed_out(torch.device(DEV))
    assert bool(torch.isnan(got).all()) if not copies else bool(torch.isnan(got[2]).all())  # (a short sequence may be done by then)
    assert bool(((got == want) | torch.isnan(got)).all())
    monkeypatch.setenv("STX_TREE_COPIES", "600")  # more than any block has
    assert torch.equal(tree_attention(q, layer, length), want) and not attention_timed_out()
    monkeypatch.delenv("STX_TREE_COPIES")
    assert torch.equal(tree_attention(q, layer, length), want) and not attention_timed_out()


def test_a_host_run_with_expired_waits_is_refused(monkeypatch):
    from test_gpu_speculative import _model, _prompt

    m = _model(dtype=F16, kv_store="int8", layers=1)
    want = m.generate_speculative(_prompt(9), 3, use_graph=False)["tokens"].tolist()
    monkeypatch.setenv("STX_TREE_COPIES", "0")
    for run in (lambda: m.generate_speculative(_prompt(9), 3, use_graph=False), lambda: m.generate(_prompt(9), 2, use_graph=False)):
        with pytest.raises(RuntimeError, match="wait"):
            run()
    monkeypatch.delenv("STX_TREE_COPIES")
    assert m.generate_speculative(_prompt(9), 3, use_graph=False)["tokens"].tolist() == want
    m.close()


@pytest.mark.parametrize("dtype,store,hd", [(F16, "same", 64), (BF16, "int8", 128), (F16, "e4m3", 128), (BF16, "same", 256), (F32, "same", 128)])
@pytest.mark.parametrize("n_seq,heads,kv,T", [(1, 3, 1, 5), (1, 24, 8, 5), (3, 8, 8, 1), (18, 8, 8, 2), (37, 4, 4, 1), (3, 8, 2, 40)])
def test_units_left_whole_and_split(dtype, store, hd, n_seq, heads, kv, T):
    """Contexts of one to ten tiles of 64 slots, alike and one apart: units that a CTA has for itself, shares of two tiles that end with
    units or inside them, and as many units as CTAs; the same bits on a second call."""
    from sparse_transformers_b200 import tree_attention
    from test_gpu_draft import attn_case, check_attention

    for tiles in (1, 2, 3, 4, 5, 8, 10) if n_seq < 10 else (2, 3, 7):
        for last in (0, 70):
            lengths = [64 * tiles - T] * (n_seq - 1) + [max(0, 64 * tiles - T - last)]
            case = attn_case(dtype, store, hd, heads, kv, T, lengths, tree="chain", seed=tiles)
            assert torch.equal(check_attention(*case), tree_attention(case[1], case[0], case[2]))


def test_positions_changed_before_the_gradient_are_refused():
    """The gradient turns back by the angles of the forward pass: positions that have moved on since are an error, not other angles."""
    from sparse_transformers_b200 import RotaryPositions

    plan = RotaryPositions(32, device=DEV)
    x = torch.randn(5, 2, 32, generator=gen(1), device=DEV).requires_grad_()
    pos = torch.arange(5, device=DEV)
    y = plan.rotate(x, pos)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = plan.rotate(x, pos)
    (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    assert_within(dx.detach(), 2 * x.detach().double(), 12 * 3.1 * 2.0 ** -24 * ref.rotate_slack(x.detach(), 16, 1.0, False))  # two rotations of 3.1 2^-24 each way, doubled
    (ddx,) = torch.autograd.grad((dx * x.detach()).sum(), x)
    assert ddx.shape == x.shape
    y = plan.rotate(x, pos)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def first_layer_keys(m, ids):
    """Keys of the first decoder layer before their rotation, as prefill forms them: [T, kv_heads, head_dim]."""
    from sparse_transformers_b200.llama_skip import rms_norm

    c, L = m.cfg, m.layers[0]
    x = rms_norm(m.embed.index_select(0, ids), L["ln1"], c.rms_eps)
    return (x @ L["wqkv"].t())[:, c.heads * c.head_dim:(c.heads + c.kv_heads) * c.head_dim].unflatten(-1, (c.kv_heads, c.head_dim))


@pytest.mark.parametrize("draft_nodes", [0, 4])
def test_a_model_has_one_rotation(draft_nodes):
    """Far from the start the prompt's keys and those of drafted tokens stand at the same angles.  A table's sine and cosine are rounded once,
    products and sum as in a rotation.  A model that neither drafts nor holds 8 bits keeps the tables that it had."""
    from sparse_transformers_b200.llama_skip import rope_tables
    from test_gpu_draft import TURN
    from test_gpu_speculative import _model, _prompt

    T = 8200
    m = _model(max_len=T + 8, layers=1, draft_nodes=draft_nodes)
    if not draft_nodes:
        assert all(torch.equal(a, b) for a, b in zip((m.cos, m.sin), rope_tables(m.cfg, DEV)))
        m.close()
        return
    ids = _prompt(T)
    m.prefill(ids)
    k, pos = first_layer_keys(m, ids), torch.arange(T, device=DEV)
    want = ref.rotate(k, pos, m.rope.frequencies, 1.0, False)
    slack = half_step(want, F32) + TURN * ref.rotate_slack(k, 32, 1.0, False)
    assert_within(m.k_cache[0, :, :T].transpose(0, 1), want, slack, "prompt")
    m.kv.layer(0).append(k.unsqueeze(0), k.unsqueeze(0), i64(0), rope=m.rope)
    assert_within(m.k_cache[0, :, :T].transpose(0, 1), want, slack, "appended")
    m.close()


@pytest.mark.parametrize("dtype,store", [(BF16, "int8"), (F16, "e4m3"), (F16, "int8")])
def test_a_prompts_keys_are_rounded_once(dtype, store):
    """An 8-bit cache holds the same codes of a key whether it came with the prompt or with a draft."""
    from test_gpu_speculative import _model, _prompt

    m = _model(dtype=dtype, kv_store=store, layers=1)
    ids = _prompt(70)
    m.prefill(ids)
    k = first_layer_keys(m, ids)
    codes, scales = m.kv.k.view(torch.uint8).clone(), m.kv.k_scale.clone()
    m.kv.layer(0).append(k.unsqueeze(0), k.unsqueeze(0), i64(0), rope=m.rope)
    assert torch.equal(m.kv.k.view(torch.uint8), codes) and torch.equal(m.kv.k_scale, scales)
    m.close()


def test_written_tensors_are_stale_for_autograd():
    """What a call writes counts as changed in place: a gradient that needs the old values is an error."""
    from sparse_transformers_b200 import KVCache, RotaryPositions, tree_attention

    plan = RotaryPositions(64, device=DEV)
    cache = KVCache(1, 2, 8, 64, dtype=F32, device=DEV)
    layer = cache.layer(0)
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.randn(1, 2, 2, 64, generator=gen(0), device=DEV)
    y, z = x.clone(), x.clone()
    for name, t, call in (("rope out", x, lambda: plan.rotate(x, i64(0, 1).view(1, 2), out=x)), ("keys", layer.k, lambda: layer.append(y, y, i64(0))),
                          ("values", cache.v, lambda: layer.append(y, y, i64(0))), ("q_out", z, lambda: layer.append(y, y, i64(0), q=y, q_out=z)),
                          ("keep", cache.k, lambda: cache.keep(i64(0), i64(0, 1).view(1, 2), i64(2))), ("out", z, lambda: tree_attention(y, layer, i64(2), out=z))):
        kept = (t * w).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
        assert y._version == 0, name
    with torch.inference_mode():  # tensors without a version
        c = KVCache(1, 2, 8, 64, dtype=F32, device=DEV)
        c.layer(0).append(y, y, i64(0))
    c.layer(0).append(y, y, i64(2))
    assert torch.equal(c.layer(0).read(i64(2), 2)[0], y.transpose(1, 2))


def test_calls_that_would_lose_a_gradient_are_refused():
    from sparse_transformers_b200 import KVCache, RotaryPositions, tree_attention

    plan = RotaryPositions(64, device=DEV)
    n, pos = i64(2), i64(0, 1).view(1, 2)
    k, v = (torch.randn(1, 2, 8, 64, generator=gen(s), device=DEV) for s in (0, 1))
    x, q = torch.randn(1, 2, 2, 64, device=DEV), torch.randn(1, 2, 2, 64, device=DEV)
    learnt = KVCache.from_tensors(k, v.clone().requires_grad_()).layer(0)
    scaled = KVCache.from_tensors(k.to(torch.int8), v.to(torch.int8), torch.ones(1, 2, 8, device=DEV), torch.ones(1, 2, 8, device=DEV, requires_grad=True), dtype=F32).layer(0)
    layer = KVCache.from_tensors(k, v).layer(0)
    for f, m in ((lambda: tree_attention(q, learnt, n), "no gradient"), (lambda: tree_attention(q, scaled, n), "no gradient"), (lambda: learnt.read(None, 4), "no gradient"),
                 (lambda: learnt.append(x, x, n), "no gradient"), (lambda: tree_attention(q, layer, n, out=torch.empty_like(q).requires_grad_()), "no gradient"),
                 (lambda: plan.rotate(x, pos, out=torch.empty_like(x).requires_grad_()), "no gradient"),
                 (lambda: layer.append(x, x, n, q=q, q_out=torch.empty_like(q).requires_grad_()), "no gradient")):
        with pytest.raises(RuntimeError, match=m):
            f()
    with torch.no_grad():  # nobody asks for a gradient
        assert torch.equal(tree_attention(q, learnt, n), tree_attention(q, layer, n))


def test_calls_that_write_what_they_read_are_refused():
    from sparse_transformers_b200 import KVCache, RotaryPositions, tree_attention

    plan = RotaryPositions(64, device=DEV)
    n, path = i64(2), i64(1, 0).view(1, 2)
    k, v = (torch.randn(1, 2, 8, 64, generator=gen(s), device=DEV) for s in (0, 1))
    x, q = torch.randn(1, 2, 2, 64, device=DEV), torch.randn(1, 2, 2, 64, device=DEV)
    cache = KVCache.from_tensors(k, v)
    layer, twice = cache.layer(0), KVCache.from_tensors(k, k)
    ones = torch.ones(2, 1, 2, 8, device=DEV)
    codes = torch.zeros(2, 1, 2, 8, 64, dtype=torch.int8, device=DEV)
    for f, m in ((lambda: twice.layer(0).append(x, x, n), "overlap"), (lambda: twice.keep(n, path, n), "overlap"),
                 (lambda: layer.append(x, x, n, q=q, q_out=x), "overlap"), (lambda: layer.append(k[:, :2, 0:2], x, n), "overlap"),
                 (lambda: layer.append(x, v[:, :2, 0:2], n), "overlap"), (lambda: layer.append(x, x, n, q=q, q_out=k.view(1, -1)[:, :256].view(1, 2, 2, 64)), "overlap"),
                 (lambda: tree_attention(q, layer, n, out=v.view(1, -1)[:, 64:320].view(1, 2, 2, 64)), "overlap"),
                 (lambda: KVCache.from_tensors(codes, codes.clone(), ones[:1].expand(2, 1, 2, 8), ones[:1].expand(2, 1, 2, 8), dtype=F16).keep(n, path, n), "more than one element|overlap|single memory")):
        with pytest.raises(RuntimeError, match=m):
            f()
    # parts of one block, q rotated in place, as a projection leaves them
    block = torch.randn(1, 2, 6, 64, generator=gen(3), device=DEV)
    want = layer.append(block[:, :, 2:4], block[:, :, 4:], n, rope=plan, q=block[:, :, :2])
    assert torch.equal(layer.append(block[:, :, 2:4], block[:, :, 4:], n, rope=plan, q=block[:, :, :2], q_out=block[:, :, :2]), want)
