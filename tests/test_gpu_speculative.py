"""Decoding from drafted tokens as a whole: the operators of one step in a row against their definitions in 64 bits, and the LlamaSkip
host's generate_speculative against its token-by-token generate.

The host is compared in fp32 with every neuron active, where both ways of decoding compute the same numbers up to sums in another
order (relative 1e-6; the gap between the two largest of the 500 logits of these random models is of the order 0.1), so that the
greedy tokens have to be equal whatever is drafted."""
import math

import numpy as np
import pytest
import torch

import draftref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(seed=2, **kw):
    from sparse_transformers_b200.llama_skip import LlamaSkipConfig, LlamaSkipModel

    base = dict(vocab=500, hidden=256, intermediate=512, layers=2, heads=4, kv_heads=2, head_dim=64, predictor_rank=32,
                density=1 - 1e-12, max_len=96, dtype=torch.float32, draft_nodes=9)
    base.update(kw)
    return LlamaSkipModel(LlamaSkipConfig(**base), DEV, seed=seed)


def _prompt(n, vocab=500, seed=0):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("store,dtype", [("same", torch.float16), ("int8", torch.bfloat16), ("e4m3", torch.float16), ("int8", torch.float32)])
def test_one_step_in_a_row(store, dtype):
    """Append (rotated), attend, verify, keep; then the next draft attends to what was kept.  Each operator is checked against its
    definition applied to what the one before it left, three ragged sequences, one of them without a draft in use."""
    from sparse_transformers_b200 import KVCache, RotaryPositions, draft_masks, tree_attention, verify_draft

    B, T, nh, kv, hd, L, V = 3, 7, 8, 2, 64, 200, 50
    g = torch.Generator(device=DEV).manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    plan = RotaryPositions(hd, theta=500000.0, device=DEV)
    cache = KVCache(B, kv, L, hd, dtype=dtype, store=store, device=DEV)
    layer = cache.layer(0)
    length = torch.tensor([0, 70, 129], device=DEV)
    layer.append(rn(B, 130, kv, hd), rn(B, 130, kv, hd), torch.zeros(B, dtype=torch.long, device=DEV), counts=length, rope=plan)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 4, 4]] * B, device=DEV)
    counts = torch.tensor([7, 0, 5], device=DEV)
    for step in range(2):
        masks, depth = draft_masks(parents)
        k, v, q = rn(B, T, kv, hd), rn(B, T, kv, hd), rn(B, T, nh, hd)
        pos = length[:, None] + depth
        q = layer.append(k, v, length, counts=counts, rope=plan, positions=pos, q=q)
        kk, vv = (t.double() for t in layer.read(None, L))
        # what was written: the rotated key within its roundings (16 bits: half a step; 8 bits: half a code and the rounding of
        # what it stands for), in rows in use
        rk = ref.rotate(k, pos, plan.frequencies, plan.factor, plan.interleaved).transpose(1, 2)
        for b in range(B):
            n = int(counts[b])
            got = kk[b, :, int(length[b]):int(length[b]) + n]
            want = rk[b, :, :n]
            eps = torch.finfo(dtype).eps
            top = want.abs().amax(-1, keepdim=True)
            code = {"same": 0.0, "int8": 0.5 / 127, "e4m3": 2.0 ** -4}[store]
            assert bool(((got - want).abs() <= (code * (top if store == "int8" else want.abs()) + 2 * eps * top + (2.0 ** -10 / 448 * top if store == "e4m3" else 0))).all())
        out = tree_attention(q, layer, length, tree=masks, counts=counts)
        m = masks.cpu().numpy().astype(np.uint64)
        want = ref.attention(q, kk, vv, length, counts, m, L)
        slack = ref.attention_slack(q, kk, vv, dtype)
        assert float((out.double() - want).abs().max()) <= slack + torch.finfo(dtype).eps / 2 * float(want.abs().max())
        tokens = torch.randint(0, V, (B, T), generator=g, device=DEV)
        target = tokens[:, [1, 3, 4, 0, 5, 2, 3]].clone()  # node 0 accepts 1, node 1 accepts 3
        target[2, 0] = tokens[2, 2]                        # the third sequence takes 2, then 4
        if bool((tokens[:, 1] == tokens[:, 2]).any()):
            tokens[:, 2] = (tokens[:, 1] + 1) % V
            target[2, 0] = tokens[2, 2]
        path, count, nxt = verify_draft(tokens, target, parents=parents, counts=counts)
        before_k, before_v = layer.read(None, L)
        cache.keep(length, path, count)
        after_k, after_v = layer.read(None, L)
        for b in range(B):
            n = int(count[b])
            p = path[b, :n].tolist()
            walk = [0] if int(counts[b]) else []
            while walk:
                child = [j for j in range(int(counts[b])) if int(parents[b, j]) == walk[-1] and int(tokens[b, j]) == int(target[b, walk[-1]])]
                if not child:
                    break
                walk.append(child[0])
            if int(counts[b]):
                assert p == walk and int(nxt[b]) == int(target[b, walk[-1]])
            l = int(length[b])
            assert torch.equal(after_k[b, :, l:l + n], before_k[b, :, [l + j for j in p]])
            assert torch.equal(after_v[b, :, l:l + n], before_v[b, :, [l + j for j in p]])
            assert torch.equal(after_k[b, :, :l], before_k[b, :, :l])
        length = length + torch.where(counts > 0, count, torch.zeros_like(count))


@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("wstd", [0.02, 0.1])
def test_greedy_tokens_do_not_depend_on_the_draft(store, use_graph, wstd):
    """wstd 0.02: the layers hardly move the residual stream and a token repeats; 0.1: attention and MLP decide the text."""
    m = _model(kv_store=store, wstd=wstd)
    prompt = _prompt(13)
    want = m.generate(prompt, 20, use_graph=use_graph)["tokens"].tolist()
    assert wstd == 0.02 or len(set(want)) > 4
    full = prompt.tolist() + want

    def own(tokens, n):
        return full[len(tokens):len(tokens) + n]

    def wrong(tokens, n):
        return [(t + 1) % 500 for t in own(tokens, n)]

    def tree(tokens, n):  # two wrong branches around the right one, which sits in every second node
        right = own(tokens, n // 2)
        ids, parents, last = [], [], -1
        for t in right:
            ids += [(t + 7) % 500, t]
            parents += [last, last]
            last = len(ids) - 1
        return ids, parents

    for draft in (own, wrong, tree, None, lambda tokens, n: []):
        r = m.generate_speculative(prompt, 20, draft, use_graph=use_graph)
        assert r["tokens"].tolist() == want
        assert r["passes"] + r["accepted"] == 19
        if draft is own:
            assert r["passes"] == 3  # 9 tokens a pass: 9 + 9 + 1
        if draft is tree:
            assert r["passes"] == 6  # 4 right nodes and the next token at 19, 14 and 9 tokens to go; then room for 3, 1 and 0 nodes
        if draft is wrong:
            assert r["accepted"] == 0
    # and token by token goes on behind a speculative run
    m.generate_speculative(prompt, 12, own, use_graph=use_graph)
    for _ in range(8):
        m.decode_step(use_graph)
    assert int(m.token) == want[19]
    m.close()


@pytest.mark.parametrize("dtype,hd,store", [(torch.float16, 64, "same"), (torch.bfloat16, 128, "int8"), (torch.bfloat16, 128, "same"), (torch.float16, 64, "e4m3")])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_graphs_replay_what_runs_eagerly(dtype, hd, store, temperature):
    """Sparse layers, 16 bits, drafts from the text itself: both ways run the same kernels in the same order."""
    prompt = torch.cat([_prompt(9)] * 3)
    runs = []
    for use_graph in (False, True):
        m = _model(dtype=dtype, head_dim=hd, kv_store=store, density=0.3, draft_nodes=12)
        runs.append([m.generate_speculative(prompt, 24, temperature=temperature, seed=4, use_graph=use_graph) for _ in range(2)])
        m.close()
    assert runs[0][0]["tokens"].tolist() == runs[1][0]["tokens"].tolist()
    assert all(0 <= t < 500 for t in runs[0][0]["tokens"].tolist())
    assert runs[0][0]["passes"] == runs[1][0]["passes"]


@pytest.mark.parametrize("wstd", [0.02, 0.1])
def test_long_context_rotary_scaling(wstd):
    """generate rotates from tables, generate_speculative forms the angles itself: the same plan, the same tokens."""
    scaling = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=32)
    m = _model(rope_scaling=scaling, wstd=wstd)
    prompt = _prompt(40, seed=3)
    want = m.generate(prompt, 16)["tokens"].tolist()
    assert m.generate_speculative(prompt, 16)["tokens"].tolist() == want
    plain = _model(wstd=wstd, rope_scaling=None)
    a, b = (x.logits.clone() for x in (m, plain) if x.prefill(prompt) is not None)
    assert float((a - b).abs().max()) > 1e-4 * float(a.abs().max())  # the scaling has an effect
    m.close()
    plain.close()


def test_refusals():
    m = _model(draft_nodes=0)
    with pytest.raises(ValueError, match="draft_nodes"):
        m.generate_speculative(_prompt(4), 4)
    m.close()
    m = _model(draft_nodes=4)
    with pytest.raises(ValueError, match="cache of"):
        m.generate_speculative(_prompt(90), 10)
    with pytest.raises(ValueError, match="temperature"):
        m.generate_speculative(_prompt(4), 4, temperature=-1.0)
    with pytest.raises(RuntimeError, match="no weight"):  # logits / 1e-45 are infinite or NaN
        m.generate_speculative(_prompt(4), 4, temperature=1e-45)
    assert len(m.generate_speculative(_prompt(4), 4)["tokens"]) == 4  # and the model is usable
    for bad in (lambda t, n: [1] * (n + 1), lambda t, n: [500] * n, lambda t, n: ([1, 2], [-1, 1]), lambda t, n: ([1, 2], [-1])):
        with pytest.raises(ValueError, match="draft"):
            m.generate_speculative(_prompt(4), 8, bad)
    m.close()
    with pytest.raises(ValueError, match="draft_nodes"):
        _model(draft_nodes=65)


def test_temperatures_share_a_graph():
    """A temperature is an input of the captured pass: near zero it gives the greedy tokens (gaps between logits of the order 0.1)."""
    m = _model(wstd=0.1)
    prompt = _prompt(13)
    want = m.generate_speculative(prompt, 16, lambda t, n: [])["tokens"].tolist()
    hot = m.generate_speculative(prompt, 16, lambda t, n: [], temperature=5.0, seed=1)["tokens"].tolist()
    graphs = len(m._draft_graphs)
    cold = m.generate_speculative(prompt, 16, lambda t, n: [], temperature=1e-4, seed=1)["tokens"].tolist()
    assert len(m._draft_graphs) == graphs and cold == want and hot != want
    m.close()


def test_captures_are_not_counted_as_decoding():
    """A pass of a new size is captured once; the decode time is that of the passes themselves, as generate's is."""
    import time

    m = _model(wstd=0.1)
    prompt = _prompt(13)
    count = iter([3, 1, 4, 2, 0, 3, 1, 4, 2, 0, 3] * 2)
    draft = lambda tokens, n: [7] * min(n, next(count))
    t = time.perf_counter()
    first = m.generate_speculative(prompt, 12, draft)
    t = time.perf_counter() - t
    assert first["capture_s"] > 0 and first["ttft_s"] + first["decode_s"] + first["capture_s"] <= t
    assert math.isclose(first["output_tokens_per_s"], 11 / first["decode_s"]) and math.isclose(first["total_tokens_per_s"], 12 / (first["ttft_s"] + first["decode_s"]))
    again = m.generate_speculative(prompt, 12, lambda tokens, n: [7] * min(n, 3))
    assert again["capture_s"] == 0.0 and again["tokens"].tolist() == first["tokens"].tolist()
    assert m.generate_speculative(prompt, 12, lambda tokens, n: [7], use_graph=False)["capture_s"] == 0.0
    m.close()


def test_graphs_of_passes_share_their_memory():
    """Each number of nodes, chain or tree, greedy or sampled, has a graph of its own; what they work in is not held once for each.
    A pass takes a workspace of 2 x 148 slots of 128 rows of 64 + 2 floats, 10 MB, so 30 graphs of their own memory would hold 300 MB."""
    m = _model(wstd=0.1, draft_nodes=9, max_len=400)
    prompt = _prompt(13)
    m.generate_speculative(prompt, 12, lambda tokens, n: [7])
    torch.cuda.synchronize()
    before, want = torch.cuda.memory_reserved(), {}
    for temperature in (0.0, 0.7):
        for kind in ("chain", "tree"):
            sizes = [8, 1, 7, 2, 6, 3, 5, 4, 0]
            for again in range(2):
                at = iter(sizes * 50)

                def draft(tokens, n):
                    ids = [(tokens[-1] + i) % 500 for i in range(min(n, next(at)))]
                    return ids if kind == "chain" else (ids, [i // 2 - 1 for i in range(len(ids))])

                r = m.generate_speculative(prompt, 300, draft, temperature=temperature, seed=1)
                assert want.setdefault((temperature, kind), r["tokens"].tolist()) == r["tokens"].tolist()  # (captured; then replayed in any order)
                sizes = sizes if temperature else sizes[::-1]
    assert len(m._draft_graphs) >= 30
    assert want[0.0, "chain"] == want[0.0, "tree"] == m.generate(prompt, 300)["tokens"].tolist()
    assert torch.cuda.memory_reserved() - before < 150 << 20
    m.close()
