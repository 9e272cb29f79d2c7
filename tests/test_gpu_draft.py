"""Rotary positions, the 8-bit cache, attention and verification of drafted tokens on the GPU, against their definitions in
64 bits (draftref.py).  Tolerances: a rounding to a type is off by eps / 2 of the value at most; what fp32 arithmetic adds is
bounded where it is used."""
import math

import numpy as np
import pytest
import torch

import draftref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
YARN = dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i64(*v):
    return torch.tensor(v, dtype=torch.long, device=DEV)


def half_step(t, dtype):
    """Largest rounding error of values t held in dtype."""
    f = torch.finfo(dtype)
    return f.eps / 2 * t.abs() + f.tiny * f.eps


def assert_within(got, want, slack, what=""):
    off = (got.double() - want.double()).abs() - slack
    assert not torch.isnan(got).any(), f"{what}: NaN"
    assert float(off.max()) <= 0, f"{what}: off by {float((got.double() - want.double()).abs().max()):.3g}, {float(off.max()):.3g} more than allowed"


# ---------------------------------------------------------------------------------- rotary positions
# Sine and cosine (times factor) are rounded to fp32 once (2^-24 of factor, the angle itself is off by 2^-53 of two million turns), the
# products and their sum to 2^-24 each: 3 * 2^-24 of (|x0| + |x1|) factor.
TURN = 3.1 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("hd,rot,layout,scaling", [(128, 128, "half", LLAMA3), (64, 64, "interleaved", None), (128, 32, "interleaved", YARN),
                                                   (96, 96, "half", dict(rope_type="linear", factor=4.0)), (80, 80, "half", None), (256, 64, "half", dict(rope_type="ntk", factor=4.0)),
                                                   (128, 10, "half", None), (6, 2, "interleaved", None), (33, 8, "half", None), (512, 512, "half", None)])
def test_rotate(dtype, hd, rot, layout, scaling):
    from sparse_transformers_b200 import RotaryPositions

    plan = RotaryPositions(hd, rotary_dim=rot, theta=10000.0, layout=layout, scaling=scaling, device=DEV)
    g = gen(hd + rot)
    for n, heads in ((1, 1), (7, 3), (130, 5)):
        x = torch.randn(n, heads, hd, generator=g, device=DEV).to(dtype)
        pos = torch.randint(0, 2_000_000, (n,), generator=g, device=DEV)
        pos[0] = 0
        for inverse in (False, True):
            want = ref.rotate(x, pos, plan.frequencies, plan.factor, plan.interleaved, inverse)
            slack = half_step(want, dtype) + TURN * ref.rotate_slack(x, rot // 2, plan.factor, plan.interleaved)
            y = plan.rotate(x, pos, inverse=inverse)
            assert_within(y, want, slack, (n, inverse))
            assert torch.equal(y[..., rot:], x[..., rot:])
            z = x.clone()
            assert plan.rotate(z, pos, inverse=inverse, out=z) is z and torch.equal(z, y)   # in place


@pytest.mark.parametrize("hd,layout", [(128, "half"), (40, "interleaved")])
def test_rotate_strided_and_batched(hd, layout):
    """Queries as a view of a projection's block, tokens of several sequences, an output with gaps, expanded positions."""
    from sparse_transformers_b200 import RotaryPositions

    plan = RotaryPositions(hd, layout=layout, device=DEV)
    g = gen(3)
    block = torch.randn(3, 5, 7 * hd, generator=g, device=DEV).to(F16)
    x = block[..., hd:5 * hd].unflatten(-1, (4, hd))
    pos = torch.randint(0, 9000, (5,), generator=g, device=DEV)
    want = plan.rotate(x.reshape(15, 4, hd).contiguous(), pos.repeat(3)).view(3, 5, 4, hd)
    assert torch.equal(plan.rotate(x, pos.expand(3, 5)), want)
    room = torch.full((3, 5, 6 * hd), 7.0, dtype=F16, device=DEV)
    view = room[..., :4 * hd].unflatten(-1, (4, hd))
    plan.rotate(x, pos.repeat(3, 1), out=view)
    assert torch.equal(view, want) and bool((room[..., 4 * hd:] == 7).all())
    odd = torch.randn(15 * 4 * hd + 1, generator=g, device=DEV).to(F16)[1:].view(15, 4, hd)   # not 16-byte aligned
    assert torch.equal(plan.rotate(odd, pos.repeat(3)), plan.rotate(odd.clone(), pos.repeat(3)))
    assert plan.rotate(x[:, :0], pos[:0].expand(3, 0)).shape == (3, 0, 4, hd)


def test_rotate_gradient():
    """Against the formula's (the transposed rotation) and against differences."""
    from sparse_transformers_b200 import RotaryPositions

    plan = RotaryPositions(32, rotary_dim=16, layout="half", scaling=YARN, device=DEV)
    g = gen(5)
    x = torch.randn(6, 2, 32, generator=g, device=DEV).requires_grad_()
    pos = torch.randint(0, 500, (6,), generator=g, device=DEV)
    up = torch.randn(6, 2, 32, generator=g, device=DEV)
    (dx,) = torch.autograd.grad((plan.rotate(x, pos) * up).sum(), x)
    want = ref.rotate(up, pos, plan.frequencies, plan.factor, False, inverse=True)
    assert_within(dx, want, half_step(want, F32) + TURN * ref.rotate_slack(up, 8, plan.factor, False))
    # the map is linear: a difference of outputs is the derivative along it, up to the roundings of 64 sums of products
    d = torch.randn(6, 2, 32, generator=g, device=DEV)
    with torch.no_grad():
        diff = ((plan.rotate(x + d, pos) - plan.rotate(x - d, pos)).double() / 2 * up.double()).sum()
    assert abs(float(diff - (dx.double() * d.double()).sum())) <= 384 * 2.0 ** -20
    # the gradient of the gradient: rotating back and forth is factor^2
    y = torch.randn(6, 2, 32, generator=g, device=DEV).requires_grad_()
    back = plan.rotate(plan.rotate(x.detach(), pos), pos, inverse=True)
    assert_within(back[..., :16], x.detach()[..., :16] * plan.factor ** 2, 2 * plan.factor * TURN * ref.rotate_slack(x.detach(), 8, 2 * plan.factor, False)[..., :16])
    with pytest.raises(RuntimeError, match="no gradient"):
        plan.rotate(y, pos, out=torch.empty_like(y))


# ---------------------------------------------------------------------------------- the cache
def check_rows(got, want, store, dtype, angle):
    """Rows read back against the values that went in (fp64); angle: allowance for the rotation."""
    slack = angle + half_step(want, dtype)
    if store != "same":
        top = want.abs().amax(-1, keepdim=True) + angle.amax(-1, keepdim=True)
        step = top / ref.MOST[store]
        # half a step of the code (e4m3: 2^-4 of the value, or half of the smallest code 2^-9), and what fp32 does to x * (M / a) and code * scale
        code = 0.5 * step if store == "int8" else torch.maximum(2.0 ** -4 * (want.abs() + angle), 2.0 ** -10 * step)
        slack = slack + code * (1 + 1e-5) + 4 * 2.0 ** -24 * top + half_step(want.abs() + code, dtype)
    assert_within(got, want, slack, store)


@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("dtype,hd,rot,layout", [(F16, 128, 128, "half"), (BF16, 64, 64, "interleaved"), (F32, 96, 48, "half"), (F16, 256, 64, "half"),
                                                 (BF16, 80, 20, "interleaved"), (F16, 40, 40, "half"), (F32, 7, 4, "half")])
def test_append_and_read(store, dtype, hd, rot, layout):
    from sparse_transformers_b200 import KVCache, RotaryPositions

    plan = RotaryPositions(hd, rotary_dim=rot, layout=layout, device=DEV)
    g = gen(hd)
    for B, T, nh, kv in ((1, 1, 1, 1), (3, 5, 6, 2), (2, 150, 4, 4)):
        rows = T + 20
        cache = KVCache(B, kv, rows, hd, dtype=dtype, store=store, device=DEV)
        layer = cache.layer(0)
        old_k, old_v = torch.randn(B, rows, kv, hd, generator=g, device=DEV).to(dtype), torch.randn(B, rows, kv, hd, generator=g, device=DEV).to(dtype)
        assert layer.append(old_k, old_v, torch.zeros(B, dtype=torch.long, device=DEV)) is None
        before = [t.clone() for t in (layer.k.view(torch.uint8), layer.v.view(torch.uint8))] + [None if t is None else t.clone() for t in (layer.k_scale, layer.v_scale)]
        qkv = torch.randn(B, T, (nh + 2 * kv) * hd, generator=g, device=DEV).to(dtype)
        q, k, v = (t.unflatten(-1, (-1, hd)) for t in qkv.split([nh * hd, kv * hd, kv * hd], -1))
        start = torch.arange(B, device=DEV) * 2 + 3
        counts = torch.tensor([T, T // 2, T - 1][:B], device=DEV)
        pos = torch.randint(0, 100000, (B, T), generator=g, device=DEV)
        out = layer.append(k, v, start, counts=counts, rope=plan, positions=pos, q=q)
        kr, vr = layer.read(start, T)
        want_q, want_k = (ref.rotate(t, pos, plan.frequencies, plan.factor, plan.interleaved) for t in (q, k))
        angle_q, angle_k = (TURN * ref.rotate_slack(t, rot // 2, plan.factor, plan.interleaved) for t in (q, k))
        for b in range(B):
            n, s = int(counts[b]), int(start[b])
            assert_within(out[b, :n], want_q[b, :n], half_step(want_q[b, :n], dtype) + angle_q[b, :n], "q") if n else None
            assert bool((out[b, n:] == 0).all())
            if n:
                check_rows(kr[b, :, :n].transpose(0, 1), want_k[b, :n], store, dtype, angle_k[b, :n])
                check_rows(vr[b, :, :n].transpose(0, 1), v[b, :n].double(), store, dtype, torch.zeros_like(v[b, :n], dtype=torch.float64))
            # all other rows are as they were, scales included
            other = torch.ones(rows, dtype=torch.bool, device=DEV)
            other[s:s + n] = False
            for now, was in zip((layer.k.view(torch.uint8), layer.v.view(torch.uint8), layer.k_scale, layer.v_scale), before):
                assert was is None or torch.equal(now[b][:, other], was[b][:, other])
        # positions default to the slots, rows without a plan are not rotated
        out2 = layer.append(k, v, start, rope=plan, q=q)
        slots = start[:, None] + torch.arange(T, device=DEV)
        want = ref.rotate(q, slots, plan.frequencies, plan.factor, plan.interleaved)
        assert_within(out2, want, half_step(want, dtype) + TURN * ref.rotate_slack(q, rot // 2, plan.factor, plan.interleaved))
        assert torch.equal(layer.append(k, v, start, q=q), q)
        check_rows(layer.read(start, T)[0].transpose(1, 2), k.double(), store, dtype, torch.zeros_like(k, dtype=torch.float64))


@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 20])
def test_append_slots_outside_the_cache(store, hd):
    from sparse_transformers_b200 import KVCache

    cache = KVCache(4, 2, 6, hd, dtype=F16, store=store, device=DEV)
    layer = cache.layer(0)
    k = torch.randn(4, 5, 2, hd, generator=gen(1), device=DEV).to(F16)
    layer.append(k, k, i64(-2, 4, 100, -(1 << 40)))
    kr, vr = layer.read(i64(-2, 4, 100, 0), 6)
    full, _ = layer.read(None, 6)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    for b, (lo, hi, s) in enumerate(((2, 5, -2), (0, 2, 4), (0, 0, 0), (0, 0, 0))):
        live = torch.zeros(6, dtype=torch.bool, device=DEV)
        for t in range(lo, hi):
            live[s + t] = True
            check_rows(full[b, :, s + t], k[b, t].double(), store, F16, zero.expand(2, hd))
        assert bool((full[b][:, ~live] == 0).all())
    assert bool((kr[0, :, :2] == 0).all()) and bool((kr[1, :, 2:] == 0).all()) and bool((kr[2] == 0).all())
    assert torch.equal(kr[0, :, 2:], full[0, :, :4]) and torch.equal(kr, vr)
    assert layer.read(None, 0)[0].shape == (4, 2, 0, hd)
    layer.append(k[:, :0], k[:, :0], i64(0, 0, 0, 0))
    layer.append(k, k, i64(0, 0, 0, 0), counts=i64(0, -3, 0, 0))
    assert torch.equal(layer.read(None, 6)[0], full)


@pytest.mark.parametrize("store", ["int8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 24])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_of_extreme_values(store, hd, dtype):
    """All zeros, one value that is not finite, the largest numbers, numbers near the smallest."""
    from sparse_transformers_b200 import KVCache

    f = torch.finfo(dtype)
    rows = torch.randn(8, hd, generator=gen(2), device=DEV).to(dtype)
    rows[0] = 0
    rows[1, 3] = float("nan")
    rows[2, hd - 1] = float("-inf")
    rows[3] = f.max
    rows[4, ::2] = -f.max
    rows[5] *= 2.0 ** -10
    rows[6] = f.smallest_normal
    rows[7] = 0
    rows[7, 1] = f.smallest_normal / 4
    layer = KVCache(1, 1, 8, hd, dtype=dtype, store=store, device=DEV).layer(0)
    layer.append(rows.view(1, 8, 1, hd), rows.view(1, 8, 1, hd), i64(0))
    k = layer.read(None, 8)[0].view(8, hd)
    assert bool((k[0] == 0).all()) and torch.isnan(k[1]).all() and torch.isnan(k[2]).all()
    for r in (3, 4, 5):
        check_rows(k[r].clamp(-f.max, f.max), rows[r].double(), store, dtype, torch.zeros(hd, dtype=torch.float64, device=DEV))
    # a scale below the smallest normal fp32 number (1.2e-38) is flushed: such rows are zeros, others as always
    for r in (6, 7):
        if float(rows[r].double().abs().max()) / ref.MOST[store] < 1.17e-38:
            assert bool((k[r] == 0).all())
        else:
            check_rows(k[r], rows[r].double(), store, dtype, torch.zeros(hd, dtype=torch.float64, device=DEV))
    assert bool(torch.isfinite(layer.k.float()).all())


def strided_cache(B, kv, rows, hd, held, order):
    """k or v in another order of memory: "token" = [n_seq, rows, kv, hd], "gap" = rows with unused room behind them."""
    if order == "token":
        return torch.zeros(B, rows, kv, hd, device=DEV).to(held).transpose(1, 2)
    if order == "gap":
        return torch.zeros(B, kv, rows, hd + 16, device=DEV).to(held)[..., :hd]
    return torch.zeros(B, kv, rows, hd, device=DEV).to(held)


@pytest.mark.parametrize("store,held", [("same", BF16), ("int8", torch.int8), ("e4m3", torch.float8_e4m3fn)])
@pytest.mark.parametrize("order", ["token", "gap"])
def test_caches_of_other_orders(store, held, order):
    from sparse_transformers_b200 import KVCache, tree_attention

    B, kv, rows, hd, T = 2, 3, 40, 64, 4
    g = gen(4)
    k, v = (torch.randn(B, 30 + T, kv, hd, generator=g, device=DEV).to(BF16) for _ in range(2))
    q = torch.randn(B, T, 6, hd, generator=g, device=DEV).to(BF16)
    got = []
    for o in ("head", order):
        s = [torch.zeros(B, kv, rows, device=DEV) for _ in range(2)] if store != "same" else [None, None]
        cache = KVCache.from_tensors(strided_cache(B, kv, rows, hd, held, o), strided_cache(B, kv, rows, hd, held, o), *s, dtype=BF16)
        layer = cache.layer(0)
        layer.append(k, v, i64(0, 5))
        cache.keep(i64(30, 35), i64(0, 2, 3).repeat(2, 1), i64(3, 2))
        got.append((*layer.read(None, rows), tree_attention(q, layer, i64(30, 35), counts=i64(3, 2))))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("store", ["same", "int8"])
@pytest.mark.parametrize("dtype,hd", [(F16, 64), (F32, 256), (BF16, 9)])
def test_keep(store, dtype, hd):
    """Accepted rows move together in all layers: ascending paths, any order, the same row twice, slots outside the cache."""
    from sparse_transformers_b200 import KVCache

    L, B, kv, rows = 3, 4, 2, 80
    cache = KVCache(B, kv, rows, hd, dtype=dtype, store=store, layers=L, device=DEV)
    g = gen(6)
    for i in range(L):
        x = torch.randn(B, rows, kv, hd, generator=g, device=DEV).to(dtype)
        cache.layer(i).append(x, -x, torch.zeros(B, dtype=torch.long, device=DEV))
    was = [cache.layer(i).read(None, rows) for i in range(L)]
    path = torch.full((B, 64), -1, dtype=torch.long, device=DEV)
    path[0, :4] = i64(0, 2, 5, 63)
    path[1, :5] = i64(3, 1, 1, 0, 7)       # any order, twice the same
    path[2] = torch.arange(64, device=DEV).flip(0)
    path[3, :3] = i64(0, 4, 9)             # slot 78 + 4 does not exist
    start, counts = i64(5, 0, 16, 78), i64(4, 5, 64, 3)
    cache.keep(start, path, counts)
    for i in range(L):
        for t, old in zip(cache.layer(i).read(None, rows), was[i]):
            want = old.clone()
            for b in range(B):
                for j in range(int(counts[b])):
                    src, dst = int(start[b] + path[b, j]), int(start[b]) + j
                    if 0 <= src < rows and 0 <= dst < rows:
                        want[b, :, dst] = old[b, :, src]
            assert torch.equal(t, want)
    cache.keep(start, path, i64(0, -1, 0, 0))


def test_draft_masks():
    from sparse_transformers_b200 import draft_masks

    r = np.random.RandomState(0)
    for B, T in ((1, 1), (5, 64), (40, 33)):
        trees = [ref.random_tree(r, T) for _ in range(B)]
        par = torch.from_numpy(np.stack([t[0] for t in trees])).to(DEV)
        masks, depth = draft_masks(par)
        want = np.stack([t[1] for t in trees]).view(np.int64)
        assert np.array_equal(masks.cpu().numpy(), want)
        assert np.array_equal(depth.cpu().numpy(), [[bin(int(x) & (2 ** 64 - 1)).count("1") - 1 for x in row] for row in want])
    masks, depth = draft_masks(i64(-1, 0, 2, 7, -5, 1).view(1, 6))   # nodes 2, 3 and 4 have no parent before them
    assert masks.tolist() == [[1, 3, 4, 8, 16, 35]] and depth.tolist() == [[0, 1, 0, 0, 0, 2]]


# ---------------------------------------------------------------------------------- attention
def attn_case(dtype, store, hd, heads, kv, T, lengths, counts=None, tree="tree", rows=None, seed=0, spread=1.0):
    from sparse_transformers_b200 import KVCache

    g, B = gen(seed), len(lengths)
    rows = rows or max(1, max(lengths) + T + 3)
    cache = KVCache(B, kv, rows, hd, dtype=dtype, store=store, device=DEV)
    k, v = (torch.randn(B, rows, kv, hd, generator=g, device=DEV).to(dtype) for _ in range(2))
    layer = cache.layer(0)
    layer.append(k, v, torch.zeros(B, dtype=torch.long, device=DEV))
    q = (spread * torch.randn(B, T, heads, hd, generator=g, device=DEV)).to(dtype)
    r = np.random.RandomState(seed)
    masks = np.stack([ref.random_tree(r, T)[1] for _ in range(B)]) if tree == "tree" else None
    return layer, q, i64(*lengths), None if counts is None else i64(*counts), masks


def held_rows(layer):
    """fp64 values of all rows, from the codes and scales themselves."""
    f = lambda t, s: t.double() if s is None else t.float().double() * s.double()[..., None]
    return f(layer.k, layer.k_scale), f(layer.v, layer.v_scale)


def check_attention(layer, q, length, counts, masks, scale=None, **kw):
    from sparse_transformers_b200 import tree_attention

    tree = None if masks is None else torch.from_numpy(np.ascontiguousarray(masks).view(np.int64)).to(DEV)
    k, v = held_rows(layer)
    want = ref.attention(q, k, v, length, counts, masks, layer.k.shape[2], scale)
    got = tree_attention(q, layer, length, tree=tree, counts=counts, scale=scale, **kw)
    assert_within(got, want, half_step(want, q.dtype) + ref.attention_slack(q, k, v, q.dtype, scale))
    if counts is not None:
        for b, n in enumerate(counts.tolist()):
            assert bool((got[b, max(0, n):] == 0).all())
    return got


@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("dtype,hd,heads,kv", [(F16, 128, 8, 2), (BF16, 64, 7, 1), (F32, 128, 4, 4), (BF16, 96, 6, 2), (F16, 256, 4, 2), (F32, 256, 8, 1), (F16, 16, 64, 1), (BF16, 208, 3, 1)])
def test_attention_shapes(store, dtype, hd, heads, kv):
    for T, lengths in ((1, [0]), (1, [1, 64, 127, 128]), (5, [200]), (13, [0, 63, 65, 300]), (64, [511, 1000]), (33, [95, 4097])):
        for tree in ("chain", "tree"):
            check_attention(*attn_case(dtype, store, hd, heads, kv, T, lengths, tree=tree, seed=hd + T))


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "int8"), (F16, "e4m3"), (F32, "same")])
def test_attention_ragged_and_long(dtype, store):
    check_attention(*attn_case(dtype, store, 64, 8, 2, 9, [20000, 3, 0, 1281, 640, 0], counts=[9, 4, 9, 0, 1, -2], seed=3))
    check_attention(*attn_case(dtype, store, 128, 3, 1, 2, [33000], seed=4))
    check_attention(*attn_case(dtype, store, 64, 2, 2, 3, [int(x) for x in np.random.RandomState(1).randint(0, 400, 70)], seed=5))
    check_attention(*attn_case(dtype, store, 64, 2, 1, 1, [7] * 1024, seed=6))


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "int8"), (F32, "e4m3"), (BF16, "same"), (F16, "e4m3")])
def test_attention_masks_lengths_and_scale(dtype, store):
    """Any mask: rows that see nothing, nodes that see later ones, bits beyond the nodes in use; lengths at and beyond the
    cache's end; another scale; very peaked scores."""
    r = np.random.RandomState(9)
    layer, q, length, counts, masks = attn_case(dtype, store, 128, 4, 2, 20, [0, 50, 130, 250], counts=[20, 11, 20, 3], seed=7, rows=256)
    masks = r.randint(0, 1 << 62, size=masks.shape).astype(np.uint64)
    masks[0, 3] = masks[0, 19] = 0
    masks[1, :] = ~np.uint64(0)
    masks[3, 0] = np.uint64(1) << np.uint64(63)
    got = check_attention(layer, q, length, counts, masks)
    assert bool((got[0, 3] == 0).all()) and bool((got[0, 19] == 0).all())
    check_attention(layer, q, i64(250, 256, 300, 1 << 50), None, masks, scale=0.25)     # nodes behind the end do not exist
    check_attention(layer, q, i64(-7, 0, 246, 255), None, None, scale=1.0)
    check_attention(layer, q, length, counts, masks, scale=0.0)
    check_attention(layer, q, length, counts, masks, scale=-0.5)
    one = masks[:1].repeat(4, 0)
    from sparse_transformers_b200 import tree_attention
    a = tree_attention(q, layer, length, tree=torch.from_numpy(masks[0].view(np.int64).copy()).to(DEV))
    b = tree_attention(q, layer, length, tree=torch.from_numpy(one.view(np.int64)).to(DEV))
    c = tree_attention(q, layer, length, tree=torch.from_numpy(masks[:1].view(np.int64)).to(DEV))
    assert torch.equal(a, b) and torch.equal(a, c)
    check_attention(*attn_case(dtype, store, 64, 4, 2, 6, [900, 2], seed=8, spread=30.0))


@pytest.mark.parametrize("dtype,store", [(F16, "same"), (BF16, "same"), (F32, "same"), (F16, "int8"), (BF16, "e4m3"), (F32, "int8")])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_ignores_what_masked_slots_hold(dtype, store, hd):
    """NaN, infinities and huge numbers behind the keys in use and in nodes that a row does not see leave it alone; the
    rows that see them are not finite, and only those."""
    from sparse_transformers_b200 import tree_attention

    T, n = 12, 150
    layer, q, length, counts, _ = attn_case(dtype, store, hd, 4, 2, T, [n, 60], counts=[T, 9], seed=11, rows=n + 64)
    parents = [-1, 0, 0, 1, 2, 2, 3, 4, 5, 6, 7, 8]     # 2, 4, 5, 7, 8, 10, 11 descend from node 2
    see = np.zeros(T, np.uint64)
    for i, p in enumerate(parents):
        see[i] = np.uint64(1 << i) | (see[p] if p >= 0 else np.uint64(0))
    masks = np.stack([see, see])
    clean = check_attention(layer, q, length, counts, masks)
    for poison in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).max):
        k, v = ([t[:, :, :].clone() for t in (layer.k, layer.k_scale) if t is not None], [t.clone() for t in (layer.v, layer.v_scale) if t is not None])
        for b, (s, c) in enumerate(((n, T), (60, 9))):
            if store == "same":
                layer.k[b, :, s + c:] = poison
                layer.v[b, :, s + c:] = poison
                layer.k[b, :, s + 2] = poison
                layer.v[b, :, s + 2, ::3] = poison
            else:
                for t in (layer.k_scale, layer.v_scale):
                    t[b, :, s + c:] = poison
                    t[b, :, s + 2] = poison
        got = tree_attention(q, layer, length, tree=torch.from_numpy(masks.view(np.int64)).to(DEV), counts=counts)
        for b, c in enumerate((T, 9)):
            for i in range(c):
                if not (int(see[i]) >> 2) & 1:
                    assert torch.equal(got[b, i], clean[b, i]), (poison, b, i)
                elif poison != poison:
                    assert torch.isnan(got[b, i]).any(), (b, i)
        for t, old in zip([t for t in (layer.k, layer.k_scale) if t is not None] + [t for t in (layer.v, layer.v_scale) if t is not None], k + v):
            t.copy_(old)
    # a value that is not finite, seen: the rows that see it get it, at its place only
    if store == "same":
        layer.v[0, 1, n + 2, 5] = float("inf")
        layer.v[0, 1, n + 5, 5] = float("-inf")
        got = tree_attention(q, layer, length, tree=torch.from_numpy(masks.view(np.int64)).to(DEV), counts=counts)
        for i in range(T):
            sees2, sees5 = (int(see[i]) >> 2) & 1, (int(see[i]) >> 5) & 1
            x = got[0, i, 2:, 5]
            assert bool(torch.isnan(x).all()) if sees2 and sees5 else bool((x == float("inf")).all()) if sees2 else torch.equal(x, clean[0, i, 2:, 5])
            assert torch.equal(got[0, i, :2], clean[0, i, :2])
            keep = [d for d in range(hd) if d != 5]
            assert torch.equal(got[0, i][:, keep], clean[0, i][:, keep])


@pytest.mark.parametrize("dtype,hd", [(F16, 128), (F32, 64)])
def test_attention_strided_streams_and_graphs(dtype, hd):
    """Queries and results as views, two calls at once on two streams, two captured calls replayed at once, another current stream."""
    from sparse_transformers_b200 import tree_attention

    layer, q, length, counts, masks = attn_case(dtype, "same", hd, 8, 2, 7, [3000, 900, 17], counts=[7, 5, 7], seed=13)
    tree = torch.from_numpy(masks.view(np.int64)).to(DEV)
    want = tree_attention(q, layer, length, tree=tree, counts=counts)
    block = torch.zeros(3, 7, 12 * hd, dtype=dtype, device=DEV)
    block[..., 2 * hd:10 * hd] = q.flatten(2)
    room = torch.full((3, 7, 9 * hd), 5.0, dtype=dtype, device=DEV)
    view = room[..., hd:].unflatten(-1, (8, hd))
    assert tree_attention(block[..., 2 * hd:10 * hd].unflatten(-1, (8, hd)), layer, length, tree=tree, counts=counts, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view, want) and bool((room[..., :hd] == 5).all())
    odd = torch.zeros(q.numel() + 1, dtype=dtype, device=DEV)[1:].view_as(q).copy_(q)   # not 16-byte aligned
    got = tree_attention(odd, layer, length, tree=tree, counts=counts)
    assert_within(got, want, 2 * (half_step(want, dtype) + ref.attention_slack(q, *held_rows(layer), dtype)))
    for _ in range(3):
        assert torch.equal(tree_attention(q, layer, length, tree=tree, counts=counts), want)   # bit for bit
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(tree_attention(q, layer, length, tree=tree, counts=counts))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for o in outs for x in o)
    graphs, results = [], []
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            results.append([tree_attention(q, layer, length, tree=tree, counts=counts) for _ in range(3)])
        graphs.append(g)
    for _ in range(5):
        for r in results:
            for x in r:
                x.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for r in results for x in r)
    # lengths are read on the device: the same graph follows them
    length.copy_(i64(100, 5, 0))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(results[0][0], tree_attention(q, layer, length, tree=tree, counts=counts))


def test_offsets_beyond_32_bits():
    """A cache whose second sequence begins 2^32 elements behind the first."""
    from sparse_transformers_b200 import KVCache, RotaryPositions, tree_attention

    far, rows, hd, kv, T = 1 << 32, 64, 128, 2, 4
    raw = torch.empty(far + 4 * kv * rows * hd, dtype=torch.int8, device=DEV)
    at = lambda o: raw[o:].as_strided((2, kv, rows, hd), (far, rows * hd, hd, 1), raw.storage_offset() + o)
    scales = [torch.zeros(2, kv, rows, device=DEV) for _ in range(2)]
    big = KVCache.from_tensors(at(0), at(2 * kv * rows * hd), *scales, dtype=F16)
    small = KVCache(2, kv, rows, hd, dtype=F16, store="int8", device=DEV)
    g = gen(1)
    k, v = (torch.randn(2, 50 + T, kv, hd, generator=g, device=DEV).to(F16) for _ in range(2))
    q = torch.randn(2, T, 4, hd, generator=g, device=DEV).to(F16)
    plan, got = RotaryPositions(hd, device=DEV), []
    for c in (big, small):
        c.layer(0).append(k, v, i64(0, 3), rope=plan)
        c.keep(i64(50, 53), i64(0, 2, 3).repeat(2, 1), i64(3, 3))
        got.append((*c.layer(0).read(i64(0, 3), 50 + T), tree_attention(q, c.layer(0), i64(50, 53))))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    del raw


# ---------------------------------------------------------------------------------- verification
def check_verify(tokens, target, uniform=None, parents=None, draft=None, counts=None):
    from sparse_transformers_b200 import verify_draft

    path, count, nxt = verify_draft(tokens, target, uniform=uniform, parents=parents, draft=draft, counts=counts)
    f = lambda t: None if t is None else t.cpu().numpy()
    x, p, u, par, q, c = f(tokens), f(target), f(uniform), f(parents), f(draft), f(counts)
    at = lambda t, b: None if t is None else t[b]
    for b in range(tokens.shape[0]):
        want, token = ref.verify(x[b], p[b], at(u, b), at(par, b), at(q, b), tokens.shape[1] if c is None else int(c[b]))
        assert path[b, :len(want)].tolist() == want and bool((path[b, len(want):] == -1).all()), b
        assert int(count[b]) == len(want) and int(nxt[b]) == token, b
    return path, count, nxt


@pytest.mark.parametrize("V", [1, 2, 127, 1000, 8192, 8193, 32001, 128256])
@pytest.mark.parametrize("B,T", [(1, 1), (3, 5), (2, 12)])
def test_verify_chain(V, B, T):
    g = gen(V + T)
    p = torch.softmax(3 * torch.randn(B, T, V, generator=g, device=DEV), -1)
    q = torch.softmax(p[:, :-1].log() + 0.5 * torch.randn(B, T - 1, V, generator=g, device=DEV), -1) if T > 1 else torch.empty(B, 0, V, device=DEV)
    for seed in range(6):
        u = torch.rand(B, T, generator=g, device=DEV)
        x = torch.zeros(B, T, dtype=torch.long, device=DEV)
        if T > 1:
            x[:, 1:] = torch.multinomial(q.flatten(0, 1), 1, generator=g).view(B, T - 1)
        if seed == 4:
            u[:] = 0.0
        if seed == 5:
            u[:] = 1.0 - 2.0 ** -24
        counts = None if seed % 2 else torch.tensor([T, 1, T - 1][:B], device=DEV)
        check_verify(x, p, u, None, q, counts)
    # sparse rows, as a filter leaves them
    cut = torch.where(p < p.amax(-1, keepdim=True) * 0.05, torch.zeros_like(p), p)
    check_verify(x, cut / cut.sum(-1, keepdim=True), u, None, q)
    check_verify(x, cut, torch.rand(B, T, generator=g, device=DEV))


@pytest.mark.parametrize("V", [3, 999, 9000, 50257])
@pytest.mark.parametrize("B,T", [(1, 2), (4, 33), (2, 64)])
def test_verify_tree(V, B, T):
    g, r = gen(V + T), np.random.RandomState(V + T)
    par = torch.from_numpy(np.stack([ref.random_tree(r, T)[0] for _ in range(B)])).to(DEV)
    p = torch.softmax(4 * torch.randn(B, T, V, generator=g, device=DEV), -1)
    for seed in range(4):
        u = torch.rand(B, T, generator=g, device=DEV)
        best = p.topk(min(3, V), -1).indices
        x = best.gather(1, par.clamp(min=0)[..., None].expand(-1, -1, best.shape[-1]))
        x = x.gather(2, torch.randint(0, best.shape[-1], (B, T, 1), generator=g, device=DEV)).squeeze(-1)   # equal siblings occur
        check_verify(x, p, u, par, None, None if seed % 2 else torch.tensor([T, 1, T - 1, 0][:B], device=DEV))
        greedy = p.argmax(-1)
        check_verify(x, greedy, None, par, None, None if seed % 2 else torch.tensor([T, 0, T // 2, -4][:B], device=DEV))
        check_verify(x, greedy)


def test_verify_odd_rows():
    """Rows without weight, with NaN or infinities, draft equal to target, tokens outside the vocabulary, u at its ends."""
    for V in (500, 20000):
        p = torch.rand(6, 3, V, generator=gen(V), device=DEV)
        q = torch.rand(6, 2, V, generator=gen(V + 1), device=DEV)
        x = torch.randint(0, V, (6, 3), generator=gen(V + 2), device=DEV)
        u = torch.rand(6, 3, generator=gen(V + 3), device=DEV)
        p[0] = 0
        p[1, :, V // 2] = float("nan")
        p[2, :, 3] = float("inf")
        q[3] = p[3, :2]
        u[3] = 1.0                # outside [0, 1): refused, and nothing is left of p - q
        x[4, 1], x[5, 2] = -1, V
        q[0] = 1.0
        check_verify(x, p, u, None, q)
        p[1, :, V // 2] = 0
        p[4, :, :] = 0
        p[4, :, V - 1] = 1e-30
        p[5, :, 1:] = 0
        check_verify(x, p, u)
        check_verify(x, p, torch.zeros_like(u))
        check_verify(x, p, torch.full_like(u, 1.0 - 2.0 ** -24))
        check_verify(x, p, torch.ones_like(u))


def test_verify_follows_the_target():
    """The emitted token after the root follows the target whatever the draft: 60000 walks over 6 tokens; a frequency's standard
    deviation is at most 0.5 / sqrt(60000) = 0.002, five of them are allowed."""
    from sparse_transformers_b200 import verify_draft

    n, V = 60000, 6
    g = gen(0)
    p = torch.tensor([0.35, 0.05, 0.0, 0.2, 0.25, 0.15], device=DEV)
    q = torch.tensor([0.05, 0.4, 0.1, 0.2, 0.05, 0.2], device=DEV)
    for mode in ("drawn", "fixed"):
        x = torch.zeros(n, 2, dtype=torch.long, device=DEV)
        x[:, 1] = torch.multinomial(q.expand(n, V), 1, generator=g).squeeze(1) if mode == "drawn" else 3
        path, count, nxt = verify_draft(x, p.expand(n, 2, V).contiguous(), uniform=torch.rand(n, 2, generator=g, device=DEV),
                                        draft=q.expand(n, 1, V).contiguous() if mode == "drawn" else None)
        first = torch.where(count == 2, x[:, 1], nxt)
        freq = torch.bincount(first, minlength=V).double() / n
        assert float((freq - p.double()).abs().max()) <= 5 * 0.5 / math.sqrt(n), mode
        assert int((first == 2).sum()) == 0


# ---------------------------------------------------------------------------------- one step, and what is refused
def test_refusals():
    from sparse_transformers_b200 import KVCache, RotaryPositions, draft_masks, tree_attention, verify_draft

    q = torch.zeros(1, 2, 4, 64, dtype=F16, device=DEV)
    layer = KVCache(1, 2, 16, 64, dtype=F16, device=DEV).layer(0)
    n = i64(3)
    for f, m in ((lambda: tree_attention(q.float(), layer, n), "the cache holds"),
                 (lambda: tree_attention(q, layer, n.int()), "int64"),
                 (lambda: tree_attention(q, layer, i64(1, 2)), "shape"),
                 (lambda: tree_attention(q.cpu(), layer, n), "CUDA only"),
                 (lambda: tree_attention(q, layer, n.cpu()), "CUDA only"),
                 (lambda: tree_attention(q[..., :3, :], layer, n), "do not divide"),
                 (lambda: tree_attention(q, layer, n, out=q), "overlap|memory"),
                 (lambda: tree_attention(torch.zeros(1, 65, 4, 64, dtype=F16, device=DEV), layer, n), "outside 1..64"),
                 (lambda: tree_attention(q, layer, n, tree=i64(1, 3, 7)), "shape"),
                 (lambda: tree_attention(q, layer, n, scale=float("nan")), "scale"),
                 (lambda: tree_attention(torch.zeros(1, 1, 2, 60, dtype=F16, device=DEV), KVCache(1, 2, 16, 60, dtype=F16, device=DEV).layer(0), n), "multiple of 8"),
                 (lambda: tree_attention(q.requires_grad_(), layer, n), "no gradient"),
                 (lambda: layer.append(q.detach(), q.detach(), n), "do not fit"),
                 (lambda: layer.append(q.detach()[:, :, :2], q.detach()[:, :, :2], n, rope=RotaryPositions(128, device=DEV)), "rotary plan"),
                 (lambda: RotaryPositions(64, device=DEV).rotate(q.detach()[0], n), "positions must have the shape"),
                 (lambda: RotaryPositions(64, device=DEV).rotate(q.detach()[0].double(), i64(0, 1)), "unsupported dtype"),
                 (lambda: draft_masks(torch.zeros(1, 65, dtype=torch.long, device=DEV)), "outside 1..64"),
                 (lambda: verify_draft(i64(0, 1).view(1, 2), torch.zeros(1, 2, 9, device=DEV)), "uniform"),
                 (lambda: verify_draft(i64(0, 1).view(1, 2), torch.zeros(1, 2, 9, dtype=F16, device=DEV), uniform=torch.zeros(1, 2, device=DEV)), "float32 probabilities"),
                 (lambda: verify_draft(i64(0, 1).view(1, 2), torch.zeros(1, 2, 400001, device=DEV), uniform=torch.zeros(1, 2, device=DEV)), "outside 1..400000"),
                 (lambda: verify_draft(i64(0, 1).view(1, 2), torch.zeros(1, 2, 9, device=DEV), uniform=torch.zeros(1, 2, device=DEV), parents=i64(-1, 0).view(1, 2), draft=torch.zeros(1, 1, 9, device=DEV)), "chain")):
        with pytest.raises(RuntimeError, match=m):
            f()
    expanded = torch.zeros(1, 2, 16, 64, dtype=F16, device=DEV).expand(3, 2, 16, 64)
    with pytest.raises(RuntimeError):
        KVCache.from_tensors(expanded, expanded.clone()).layer(0).append(torch.zeros(3, 1, 2, 64, dtype=F16, device=DEV), torch.zeros(3, 1, 2, 64, dtype=F16, device=DEV), i64(0, 0, 0))
