"""Drafted-token operators without a GPU: argument checks of the C ABI (made before anything is launched) and the rotary plans."""
import ctypes
import math

import pytest
import torch


def _structs(**kw):
    from sparse_transformers_b200 import _capi as C

    f = dict(k=16, v=16, k_scale=None, v_scale=None, seq_stride=16 * 64, head_stride=8 * 64, slot_stride=64, scale_seq_stride=0, scale_head_stride=0,
             max_len=8, n_seq=2, n_kv_heads=2, head_dim=64, store=C.STORE_SAME, dtype=C.F16)
    f.update(kw)
    return C, C.KV(**f), C.Heads(16, 256, 128, 64), C.Rotary(16, 64, 0, 1.0)


def _refused(C, rc, text, status=None):
    assert rc == (C.ERR_INVALID_ARG if status is None else status)
    assert text in C.last_error(), C.last_error()


@pytest.mark.parametrize("field,text", [(dict(k=None), "null cache"), (dict(dtype=7), "bad dtype"), (dict(store=5), "bad store"), (dict(store=1), "needs k_scale"),
                                        (dict(n_seq=0), "empty"), (dict(max_len=0), "empty"), (dict(max_len=1 << 40), "too large"), (dict(head_dim=257), "outside 1..256"),
                                        (dict(slot_stride=63), "strides"), (dict(seq_stride=-1), "strides")])
def test_bad_caches_are_refused_everywhere(field, text):
    C, kv, h, rot = _structs(**field)
    p = ctypes.byref
    _refused(C, C.lib.stx_kv_append(p(kv), p(h), p(h), 1, 16, None, None, None, 0, None, None, 0, None), text)
    _refused(C, C.lib.stx_kv_read(p(kv), None, 1, 16, 16, None), text)
    _refused(C, C.lib.stx_kv_keep(p(kv), 1, 0, 0, 16, 16, 4, 4, 16, None), text)
    _refused(C, C.lib.stx_tree_attention(p(kv), p(h), p(h), 1, 4, 1.0, 16, None, None, 0, 16, None), text)


def test_bad_calls_are_refused():
    C, kv, h, rot = _structs()
    p, lib, n = ctypes.byref, C.lib, ctypes.c_size_t()
    _refused(C, lib.stx_rope(None, p(h), 1, 1, 1, 64, 16, 0, p(rot), 0, C.F16, None), "null x")
    _refused(C, lib.stx_rope(p(h), p(h), 1, 1, 1, 64, None, 0, p(rot), 0, C.F16, None), "null pointer")
    _refused(C, lib.stx_rope(p(h), p(h), 1, 1, 1, 62, 16, 0, p(rot), 0, C.F16, None), "rotary_dim 64 of a head of 62")
    _refused(C, lib.stx_rope(p(h), p(h), 1, 1, 1, 2048, 16, 0, p(rot), 0, C.F16, None), "bad shape")
    _refused(C, lib.stx_rope(p(h), p(h), 1, 1, 1, 64, 16, 0, p(C.Rotary(16, 7, 0, 1.0)), 0, C.F16, None), "rotary_dim 7")
    _refused(C, lib.stx_rope(p(h), p(h), 1, 1, 1, 64, 16, 0, p(rot), 0, 9, None), "bad dtype")
    assert lib.stx_rope(p(h), p(h), 0, 5, 1, 64, 16, 0, p(rot), 0, C.F16, None) == C.OK      # nothing to do
    _refused(C, lib.stx_kv_append(p(kv), p(h), p(h), 1, None, None, None, None, 0, None, None, 0, None), "null start")
    _refused(C, lib.stx_kv_append(p(kv), None, p(h), 1, 16, None, None, None, 0, None, None, 0, None), "null k")
    _refused(C, lib.stx_kv_append(p(kv), p(h), p(h), 1, 16, None, None, None, 0, p(h), None, 4, None), "null q_out")
    _refused(C, lib.stx_kv_append(p(kv), p(h), p(h), 1, 16, None, None, None, 0, p(h), p(h), 0, None), "n_heads")
    _refused(C, lib.stx_kv_append(p(kv), p(C.Heads(16, -1, 1, 1)), p(h), 1, 16, None, None, None, 0, None, None, 0, None), "negative stride")
    _refused(C, lib.stx_kv_read(p(kv), None, -1, 16, 16, None), "out of range")
    _refused(C, lib.stx_kv_read(p(kv), None, 1, None, 16, None), "null output")
    _refused(C, lib.stx_kv_keep(p(kv), 1, 0, 0, 16, 16, 4, 65, 16, None), "longer than 64")
    _refused(C, lib.stx_kv_keep(p(kv), 0, 0, 0, 16, 16, 4, 4, 16, None), "layers")
    _refused(C, lib.stx_draft_masks(16, 1, 65, 16, 16, None), "outside 1..64")
    _refused(C, lib.stx_draft_masks(None, 1, 5, 16, 16, None), "null")
    at = lambda **k: lib.stx_tree_attention(p(k.get("kv", kv)), p(h), p(h), k.get("T", 1), k.get("nh", 4), k.get("scale", 1.0), k.get("len", 16), None, None, 0, k.get("ws", 16), None)
    _refused(C, at(T=0), "outside 1..64")
    _refused(C, at(T=65), "outside 1..64")
    _refused(C, at(nh=5), "do not divide")
    _refused(C, at(nh=130), "64 at most")
    _refused(C, at(len=None), "null")
    _refused(C, at(ws=None), "null")
    _refused(C, at(ws=24), "aligned")
    _refused(C, at(scale=float("inf")), "scale")
    _refused(C, at(kv=_structs(n_seq=1025)[1]), "1024 at most")
    _refused(C, at(kv=_structs(head_dim=60)[1]), "multiple of 8")
    _refused(C, at(kv=_structs(head_dim=40, store=1, k_scale=16, v_scale=16)[1]), "not a multiple of 16")
    _refused(C, lib.stx_tree_attention_workspace_bytes(65, 4, 2, 64, C.F16, p(n)), "outside 1..64")
    assert lib.stx_tree_attention_workspace_bytes(64, 32, 8, 128, C.F16, p(n)) == C.OK and n.value > 0
    v = lambda **k: lib.stx_verify_draft(16, k.get("par"), k.get("p", 16), k.get("t"), k.get("q"), k.get("u", 16), None, 1, k.get("T", 3), k.get("V", 100), 16, 16, 16, None)
    _refused(C, v(p=None), "one of them")
    _refused(C, v(t=16), "one of them")
    _refused(C, v(u=None), "need uniform")
    _refused(C, v(p=None, t=16), "neither")
    _refused(C, v(q=16, par=16), "chain")
    _refused(C, v(V=0), "outside 1..400000")
    _refused(C, v(V=400001), "outside 1..400000")
    _refused(C, v(T=65), "outside 1..64")


def test_rotary_frequencies():
    from sparse_transformers_b200 import RotaryPositions, rotary_frequencies

    w, f = rotary_frequencies(8, 10000.0)
    assert f == 1.0 and w == [10000.0 ** (-i / 4) for i in range(4)]
    assert rotary_frequencies(8, 10000.0, dict(rope_type="linear", factor=4.0))[0] == [x / 4 for x in w]
    assert rotary_frequencies(8, 10000.0, dict(rope_type="default")) == (w, 1.0)
    ntk, _ = rotary_frequencies(8, 10000.0, dict(rope_type="ntk", factor=4.0))
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], w[-1] / 4, rel_tol=1e-12)      # the slowest pair is slowed by factor
    big, _ = rotary_frequencies(128, 500000.0)
    l3, f = rotary_frequencies(128, 500000.0, dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192))
    assert f == 1.0
    for a, b in zip(big, l3):
        turns = 8192 * a / (2 * math.pi)
        assert math.isclose(b, a if turns >= 4 else a / 8 if turns <= 1 else a * ((turns - 1) / 3 + (4 - turns) / 3 / 8), rel_tol=1e-12)
    yarn, f = rotary_frequencies(128, 10000.0, dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096))
    base, _ = rotary_frequencies(128, 10000.0)
    assert math.isclose(f, 0.1 * math.log(16.0) + 1.0)
    lo = math.floor(128 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    hi = math.ceil(128 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    for i, (a, b) in enumerate(zip(base, yarn)):
        share = min(1.0, max(0.0, (i - lo) / (hi - lo)))
        assert math.isclose(b, a * (1 - share) + a / 16 * share, rel_tol=1e-12)
    assert rotary_frequencies(128, 1e4, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=4096, attention_factor=1.5))[1] == 1.5
    for bad in (lambda: rotary_frequencies(7), lambda: rotary_frequencies(0), lambda: rotary_frequencies(8, -1.0), lambda: rotary_frequencies(8, 1e4, dict(rope_type="linear", factor=0.0)),
                lambda: rotary_frequencies(8, 1e4, dict(rope_type="what", factor=2.0)), lambda: rotary_frequencies(8, 1e4, dict(rope_type="yarn", factor=2.0)),
                lambda: RotaryPositions(64, rotary_dim=66, device="cpu"), lambda: RotaryPositions(64, layout="other", device="cpu"),
                lambda: RotaryPositions(64, rotary_dim=32, device="cpu").tables(4)):
        with pytest.raises(ValueError):
            bad()
    plan = RotaryPositions(16, device="cpu")
    cos, sin = plan.tables(100)
    a = torch.arange(100, dtype=torch.float64)[:, None] * torch.tensor(plan.frequencies, dtype=torch.float64)
    assert float((cos[:, :8].double() - a.cos()).abs().max()) <= 2.0 ** -23 and torch.equal(sin[:, :8], sin[:, 8:])


def test_cpu_tensors_and_bad_caches_are_refused():
    from sparse_transformers_b200 import KVCache, RotaryPositions, draft_masks, tree_attention, verify_draft

    cache = KVCache(1, 2, 8, 64, device="cpu", store="int8", layers=2)
    assert cache.max_len == 8 and cache.layer(1).k.dtype == torch.int8 and cache.layer(1).k_scale.shape == (1, 2, 8)
    n = torch.zeros(1, dtype=torch.long)
    for f in (lambda: tree_attention(torch.zeros(1, 1, 2, 64), cache.layer(0), n), lambda: cache.layer(0).append(torch.zeros(1, 1, 2, 64), torch.zeros(1, 1, 2, 64), n),
              lambda: cache.layer(0).read(None, 1), lambda: cache.keep(n, n.view(1, 1), n), lambda: draft_masks(n.view(1, 1)),
              lambda: verify_draft(n.view(1, 1), n.view(1, 1)), lambda: RotaryPositions(64, device="cpu").rotate(torch.zeros(1, 2, 64), n)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    for f in (lambda: KVCache(1, 1, 1, 8, dtype=torch.float64, device="cpu"), lambda: KVCache(1, 1, 1, 8, store="int4", device="cpu"),
              lambda: KVCache.from_tensors(torch.zeros(1, 2, 3), torch.zeros(1, 2, 3)), lambda: KVCache.from_tensors(*[torch.zeros(1, 1, 1, 8, dtype=torch.int8)] * 2)):
        with pytest.raises(ValueError):
            f()


def test_prompt_lookup():
    from sparse_transformers_b200.llama_skip import prompt_lookup

    assert prompt_lookup([1, 2, 3, 9, 1, 2, 3], 2) == [9, 1]
    assert prompt_lookup([1, 2, 3, 9, 1, 2, 3], 0) == []
    assert prompt_lookup([4, 5, 6], 3) == []
    assert prompt_lookup([7], 3) == [] and prompt_lookup([], 3) == []
    assert prompt_lookup([8, 1, 5, 8, 2, 6, 8], 1) == [2]             # the latest occurrence
    assert prompt_lookup([8, 8], 4) == [8]


@pytest.mark.parametrize("scaling,text", [
    (dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096, mscale=1.0, mscale_all_dim=0.8), "mscale"),
    (dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096, truncate=False), "truncate"),
    (dict(rope_type="linear", factor=4.0, rope_theta=5e5), "rope_theta"), (dict(rope_type="default", factor=4.0), "factor"),
    (dict(factor=4.0), "factor"), (dict(rope_type="linear"), "needs factor"), (dict(rope_type="ntk"), "needs factor"),
    (dict(rope_type="yarn", original_max_position_embeddings=4096), "needs factor"),
    (dict(rope_type="llama3", factor=8.0, high_freq_factor=4.0, original_max_position_embeddings=8192), "needs low_freq_factor"),
    (dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, original_max_position_embeddings=8192), "needs high_freq_factor"),
    (dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0), "needs original_max_position_embeddings"),
    (dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=0), "must be positive"), (dict(rope_type="longrope", factor=4.0), "unknown")])
def test_rotary_scalings_that_would_be_taken_for_others_are_refused(scaling, text):
    """A key that changes the result and is not known, or one that is missing, is an error and not another rotation."""
    from sparse_transformers_b200 import rotary_frequencies

    with pytest.raises(ValueError, match=text):
        rotary_frequencies(64, 10000.0, scaling)
    if scaling.get("rope_type") == "yarn":  # the pairs' places are counted in logarithms of theta
        with pytest.raises(ValueError, match="theta"):
            rotary_frequencies(64, 1.0, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096))


def test_rotary_scalings_as_configurations_spell_them():
    from sparse_transformers_b200 import rotary_frequencies

    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)
    assert rotary_frequencies(64, 1e4, dict(yarn, type="yarn", beta_fast=32, beta_slow=1, attention_factor=None, truncate=True)) == rotary_frequencies(64, 1e4, yarn)
    assert rotary_frequencies(64, 1e4, dict(yarn, beta_fast=None, beta_slow=None)) == rotary_frequencies(64, 1e4, yarn)
    assert rotary_frequencies(64, 1e4, dict(type="linear", factor=2, original_max_position_embeddings=4096)) == rotary_frequencies(64, 1e4, dict(rope_type="linear", factor=2.0))
    assert rotary_frequencies(64, 1e4, dict(rope_type="default")) == rotary_frequencies(64, 1e4) == rotary_frequencies(64, 1e4, {})


def test_written_tensors_are_named_in_the_schemas():
    """A program that is cleaned up by its operators' schemas keeps the calls that only write."""
    import sparse_transformers_b200  # noqa: F401

    ops = torch.ops.sparse_mlp
    writes = lambda op: [a.name for a in op._schema.arguments if a.alias_info is not None and a.alias_info.is_write]
    cache = ["k_cache", "v_cache", "k_scale", "v_scale"]
    assert writes(ops.kv_append.default) == cache and writes(ops.kv_keep.default) == cache and writes(ops.kv_append.out) == cache + ["q_out"]
    assert writes(ops.rope.out) == ["out"] and writes(ops.tree_attention.out) == ["out"]
    assert not writes(ops.rope.default) and not writes(ops.tree_attention.default) and not writes(ops.kv_read.default)
    g = torch.fx.Graph()
    k, v, x, n = (g.placeholder(name) for name in ("k", "v", "x", "n"))
    g.call_function(ops.kv_append.default, (k, v, None, None, x, x, n, None, None, False, 1.0, None, None))
    g.call_function(ops.kv_keep.default, (k, v, None, None, 1, n, n, n))
    g.call_function(ops.rope.out, (x, n, n, False, 1.0, False), dict(out=x))
    g.call_function(ops.tree_attention.out, (x, k, v, None, None, n, None, None, None), dict(out=x))
    g.output(n)
    g.eliminate_dead_code()
    assert sum(node.op == "call_function" for node in g.nodes) == 4
