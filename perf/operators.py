"""Operators of decoding from drafted tokens, as they are measured: a plain form of each and the package's own call.

  rope     rotary positions of queries or keys (half and interleaved layouts, part of the head, scaled for long contexts)
  append   the cache is written: keys rotated, keys and values held in 16 or 8 bits, the rows read back
  read     a stretch of an 8-bit cache read back
  attn     attention of drafted tokens (a chain or a tree) over the cache
  verify   drafted tokens against the target's distributions, from given random numbers

Sequences of a ragged batch have lengths and counts that follow from their index, so the work of a case is known without
its inputs.  Everything else comes from the seed.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
MOST = {"int8": 127.0, "e4m3": 448.0}


# ---------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a decoded token of eight requests, queries only: nothing but latency
        dict(name="rope-decode-fp16", kind="rope", N=8, heads=32, hd=128, rot=128, layout="half", scaling="llama3", theta=500000.0, factor=8.0, orig=8192, far=131072, inverse=False, dtype="fp16"),
        # a prompt's queries and keys, a quarter of the head rotated in pairs, stretched sixteen times, turned back
        # (the gradient of a rotation); odd number of tokens
        dict(name="rope-partial-bf16-8191", kind="rope", N=8191, heads=40, hd=128, rot=32, layout="interleaved", scaling="yarn", theta=10000.0, factor=16.0, orig=4096, far=65536, inverse=True, dtype="bf16"),
        # one token for each of eight requests into an 8-bit cache
        dict(name="append-decode-int8", kind="append", B=8, T=1, heads=32, kv=8, hd=128, rot=128, layout="half", scaling="none", theta=500000.0, factor=1.0, orig=8192, far=4096, ragged=True, store="int8", dtype="fp16"),
        # a tree of 13 nodes for three requests, cache in the model's type, interleaved pairs
        dict(name="append-tree-bf16", kind="append", B=3, T=13, heads=16, kv=4, hd=64, rot=64, layout="interleaved", scaling="none", theta=10000.0, factor=1.0, orig=4096, far=1000, ragged=True, store="same", dtype="bf16"),
        # two prompts of 4096 tokens into a cache of 8-bit floats
        dict(name="append-prompt-e4m3", kind="append", B=2, T=4096, heads=32, kv=8, hd=128, rot=128, layout="half", scaling="linear", theta=10000.0, factor=4.0, orig=4096, far=0, ragged=False, store="e4m3", dtype="bf16"),
        # a cached prompt handed to a part that wants 16 bits
        dict(name="read-int8-16k", kind="read", B=2, kv=8, hd=128, n=16384, store="int8", dtype="fp16"),
        # a chain of five drafted tokens early in a conversation, 3B shape: latency
        dict(name="attn-chain5-fp16-ctx200", kind="attn", B=1, T=5, heads=24, kv=8, hd=128, ctx=200, ragged=False, tree=False, store="same", dtype="fp16"),
        # a serving batch of 16 requests, trees of eight nodes, int8 cache, uneven lengths
        dict(name="attn-b16-tree8-int8", kind="attn", B=16, T=8, heads=32, kv=8, hd=128, ctx=6000, ragged=True, tree=True, store="int8", dtype="bf16"),
        # one token at a time over a cache of 8-bit floats, heads of 64, 7 query heads to a cache head
        dict(name="attn-b5-t1-e4m3-hd64", kind="attn", B=5, T=1, heads=28, kv=4, hd=64, ctx=9001, ragged=True, tree=False, store="e4m3", dtype="fp16"),
        # a full tree of 64 nodes behind 32768 tokens: the largest call
        dict(name="attn-tree64-bf16-32k", kind="attn", B=1, T=64, heads=32, kv=8, hd=128, ctx=32768, ragged=False, tree=True, store="same", dtype="bf16"),
        # 32 requests, chains of five drafted tokens with the draft's own distributions, large vocabulary
        dict(name="verify-chain-b32-128k", kind="verify", B=32, T=6, V=128256, mode="chain", ragged=True),
        # one request, a tree of 32 fixed candidates
        dict(name="verify-tree32-32k", kind="verify", B=1, T=32, V=32000, mode="tree", ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges, no larger than the largest listed one."""
    c, most = _draw(rng), max(work(c)["bytes"] for c in listed())
    size = {"rope": "N", "read": "n", "append": "T"}.get(c["kind"])
    while size and work(c)["bytes"] > most:
        c[size] = c[size] * 2 // 3
    return c


def _draw(rng):
    kind = rng.choice(["rope", "append", "read", "attn", "attn", "attn", "verify", "verify"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"])
    if kind == "verify":
        V = _log(rng, 1000, 152064)
        mode = rng.choice(["chain", "tree", "tree", "greedy"])
        T = rng.randint(1, 12) if mode == "chain" else rng.randint(1, 64)
        B = max(1, min(_log(rng, 1, 48), 25_000_000 // (T * V)))
        return dict(kind=kind, B=B, T=T, V=V, mode=mode, ragged=rng.random() < 0.5)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
    hd = rng.choice([64, 64, 96, 128, 128, 128, 256])
    store = rng.choice(["same", "int8", "e4m3"])
    if kind == "read":
        B = rng.randint(1, 6)
        return dict(kind=kind, B=B, kv=kv, hd=hd, n=_log(rng, 1, max(1, 33_000_000 // (B * kv * hd))), store=store, dtype=dtype)
    if kind == "attn":
        if dtype == "fp32":  # the 32-bit form serves checking runs: short
            T, B, ctx = _log(rng, 1, 16), _log(rng, 1, 8), _log(rng, 1, 4000)
        else:
            T, B, ctx = _log(rng, 1, 64), _log(rng, 1, 32), _log(rng, 1, 32768)
        ctx = min(ctx, (8 * 32768 * 128) // (B * kv * hd), (64 * 32 * 32768 * 128) // (B * T * heads * hd))
        return dict(kind=kind, B=B, T=T, heads=heads, kv=kv, hd=hd, ctx=max(1, ctx), ragged=rng.random() < 0.6, tree=rng.random() < 0.6, store=store, dtype=dtype)
    scaling = rng.choice(["none", "linear", "ntk", "llama3", "yarn"])
    rot = rng.choice([hd, hd, hd // 2, hd // 4, 10])
    about = dict(rot=rot, layout=rng.choice(["half", "interleaved"]), scaling=scaling, theta=rng.choice([10000.0, 500000.0, 1000000.0]), factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 16.0]), orig=rng.choice([4096, 8192]), far=_log(rng, 1, 1000000))
    if kind == "rope":
        return dict(kind=kind, N=_log(rng, 1, max(1, 40_000_000 // (heads * hd))), heads=heads, hd=hd, inverse=rng.random() < 0.4, dtype=dtype, **about)
    B = _log(rng, 1, 16)
    about["far"] = _log(rng, 1, 2000)
    if dtype == "fp32":  # a checking run keeps its cache in 32 bits too
        store = "same"
    return dict(kind=kind, B=B, T=_log(rng, 1, max(1, 8192 * 48 * 128 // (B * (heads + 2 * kv) * hd))) if rng.random() < 0.5 else rng.randint(1, 64), heads=heads, kv=kv, hd=hd, ragged=rng.random() < 0.6, store=store, dtype=dtype, **about)


# ---------------------------------------------------------------------------------- what follows from a case alone
def _lengths(c):
    """Prefix lengths of the sequences: from an eighth of the context to all of it."""
    B, n = c["B"], c["ctx"]
    return [n - (n - n // 8) * b // max(1, B - 1) if c["ragged"] else n for b in range(B)]


def _counts(c):
    """Nodes in use: a ragged batch leaves some of the T behind in every second and third sequence."""
    return [max(1, c["T"] - b % 3) if c["ragged"] else c["T"] for b in range(c["B"])]


def _starts(c):
    return [max(0, c["far"] - 37 * b) if c["ragged"] else c["far"] for b in range(c["B"])]


def work(case):
    c = case
    if c["kind"] == "rope":
        return {"bytes": 2 * c["N"] * c["heads"] * c["hd"] * SIZE[c["dtype"]] + 8 * c["N"], "flops": 3 * c["N"] * c["heads"] * c["rot"]}
    if c["kind"] == "verify":
        if c["mode"] == "greedy":
            return {"bytes": c["B"] * (8 * 3 * c["T"] + 16 + 8 * c["T"]), "flops": c["B"] * c["T"]}
        rows = c["B"] * (2 if c["mode"] == "chain" and c["T"] > 1 else 1)  # one token is drawn at least, from a row (less another)
        return {"bytes": 4 * rows * c["V"] + 8 * 4 * c["B"] * c["T"], "flops": 2 * rows * c["V"]}
    s, row = SIZE[c["dtype"]], (c["hd"] + 4 if c["store"] != "same" else c["hd"] * SIZE[c["dtype"]])
    if c["kind"] == "read":
        return {"bytes": 2 * c["B"] * c["kv"] * c["n"] * (row + c["hd"] * s), "flops": 2 * c["B"] * c["kv"] * c["n"] * c["hd"]}
    if c["kind"] == "append":  # the inputs, the rotated queries, the rows once written and once read, the rows handed back
        n = sum(_counts(c))
        moved = n * ((2 * c["heads"] + 2 * c["kv"]) * c["hd"] * s + 4 * c["kv"] * row) + 2 * c["B"] * c["T"] * c["kv"] * c["hd"] * s
        return {"bytes": moved, "flops": 3 * n * (c["heads"] + c["kv"]) * c["rot"] + 4 * n * c["kv"] * c["hd"]}
    keys = sum(l + n for l, n in zip(_lengths(c), _counts(c)))
    pairs = sum((l + 1) * n for l, n in zip(_lengths(c), _counts(c)))  # a node sees the prefix and itself at least
    return {"bytes": 2 * c["kv"] * keys * row + 2 * sum(_counts(c)) * c["heads"] * c["hd"] * s, "flops": 4 * c["hd"] * c["heads"] * pairs}


# ---------------------------------------------------------------------------------- inputs
def _gen(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + salt) % (1 << 62))


def _rn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _i64(values):
    return torch.tensor(values, dtype=torch.long, device="cuda")


def _keys(g, *shape):
    """Keys as models have them: some channels are several times as large as others."""
    return _rn(g, *shape) * torch.exp(0.5 * _rn(g, shape[-1]))


def _hold(x, store, dtype):
    """Rows as a cache holds them: (what is stored, the scale of each row or None)."""
    if store == "same":
        return x.to(dtype), None
    x = x.float()
    most = MOST[store]
    top = x.abs().amax(-1, keepdim=True)
    codes = x * torch.where(top > 0, most / top, torch.zeros_like(top))
    codes = torch.round(codes).to(torch.int8) if store == "int8" else codes.to(torch.float8_e4m3fn)
    return codes, (top / most).squeeze(-1)


def _held(codes, scale):
    """The values that stored rows stand for, in 32 bits."""
    return codes.float() if scale is None else codes.float() * scale.unsqueeze(-1)


def _rope_plan(c):
    """(angle per position of each pair in 64 bits, factor of the result)"""
    rot, theta, f, orig = c["rot"], c["theta"], c["factor"], c["orig"]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    if c["scaling"] == "ntk" and rot > 2:
        theta = theta * f ** (rot / (rot - 2))
    w = theta ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        return w / f, 1.0
    if c["scaling"] == "llama3":
        turns = orig * w / (2 * math.pi)  # turns within the trained context: under 1 stretched, over 4 left alone
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return w * (keep + (1 - keep) / f), 1.0
    if c["scaling"] == "yarn":
        at = lambda n: rot * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(theta))  # the pair that turns n times in it
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return w * (1 - ramp + ramp / f), 0.1 * math.log(f) + 1.0
    return w, 1.0


def _scaling(c):
    """The same as RotaryPositions takes it."""
    if c["scaling"] == "none":
        return None
    s = dict(rope_type=c["scaling"], factor=c["factor"], original_max_position_embeddings=c["orig"])
    if c["scaling"] == "llama3":
        s.update(low_freq_factor=1.0, high_freq_factor=4.0)
    return s


def _parents(c, seed):
    """parents [B,T] (node 0 is the root) and what each node sees: itself and its ancestors, as bits."""
    r = np.random.RandomState(seed % (1 << 31))
    B, T = c["B"], c["T"]
    par = np.full((B, T), -1, np.int64)
    sees = np.zeros((B, T), np.uint64)
    for b in range(B):
        for i in range(T):
            par[b, i] = (i - 1) if not c.get("tree", True) or i == 0 else r.randint(max(0, i - 6), i)
            sees[b, i] = np.uint64(1 << i) | (sees[b, par[b, i]] if i else np.uint64(0))
    return _i64(par), torch.from_numpy(sees.view(np.int64)).cuda()


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "verify":
        return _prepare_verify(c, seed, g)
    dt = DTYPES[c["dtype"]]
    s = dict(case=c)
    if c["kind"] in ("rope", "append"):
        s["w"], s["f"] = _rope_plan(c)
    if c["kind"] == "rope":
        s["x"] = _rn(g, c["N"], c["heads"], c["hd"]).to(dt)
        s["pos"] = torch.randint(0, max(1, c["far"]), (c["N"],), generator=g, device="cuda")
    elif c["kind"] == "append":
        B, T, nh, kv, hd = c["B"], c["T"], c["heads"], c["kv"], c["hd"]
        qkv = torch.cat([1.5 * _rn(g, B, T, nh * hd), _keys(g, B, T, kv, hd).flatten(2), _rn(g, B, T, kv * hd)], -1).to(dt)
        q, k, v = qkv.split([nh * hd, kv * hd, kv * hd], -1)  # as a projection leaves them: views of one block
        s["q"], s["k"], s["v"] = q.unflatten(-1, (nh, hd)), k.unflatten(-1, (kv, hd)), v.unflatten(-1, (kv, hd))
        s["start"], s["counts"] = _i64(_starts(c)), _i64(_counts(c))
        rows = c["far"] + T + 5
        s["kc"], s["ks"] = _hold(_rn(g, B, kv, rows, hd), c["store"], dt)
        s["vc"], s["vs"] = _hold(_rn(g, B, kv, rows, hd), c["store"], dt)
        # nodes of a tree stand at their depth: positions are an input
        s["pos"] = s["start"][:, None] + torch.minimum(torch.arange(T, device="cuda"), torch.randint(0, T, (B, T), generator=g, device="cuda"))
    elif c["kind"] == "read":
        s["kc"], s["ks"] = _hold(_keys(g, c["B"], c["kv"], c["n"] + 3, c["hd"]), c["store"], dt)
        s["vc"], s["vs"] = _hold(_rn(g, c["B"], c["kv"], c["n"] + 3, c["hd"]), c["store"], dt)
        s["start"] = _i64([b % 4 for b in range(c["B"])])
    else:
        rows = c["ctx"] + c["T"] + 3
        s["q"] = (1.5 * _rn(g, c["B"], c["T"], c["heads"], c["hd"])).to(dt)
        s["kc"], s["ks"] = _hold(_keys(g, c["B"], c["kv"], rows, c["hd"]), c["store"], dt)
        s["vc"], s["vs"] = _hold(_rn(g, c["B"], c["kv"], rows, c["hd"]), c["store"], dt)
        s["length"], s["counts"] = _i64(_lengths(c)), _i64(_counts(c))
        s["parents"], s["sees"] = _parents(c, seed)
    if own:
        from sparse_transformers_b200 import KVCache, RotaryPositions

        if "w" in s:
            s["rope"] = RotaryPositions(c["hd"], rotary_dim=c["rot"], theta=c["theta"], layout=c["layout"], scaling=_scaling(c), device="cuda")
        if "kc" in s:
            s["cache"] = KVCache.from_tensors(s["kc"], s["vc"], s["ks"], s["vs"], dtype=dt)
    return s


def _prepare_verify(c, seed, g):
    B, T, V, mode = c["B"], c["T"], c["V"], c["mode"]
    s = dict(case=c, counts=_i64(_counts(c)))
    s["parents"], s["sees"] = _parents(dict(c, tree=mode != "chain"), seed)
    par = s["parents"].clamp(min=0)
    if mode == "greedy":
        s["target"] = torch.randint(0, V, (B, T), generator=g, device="cuda")
        hit = torch.rand(B, T, generator=g, device="cuda") < 0.7
        s["tokens"] = torch.where(hit, s["target"].gather(1, par), torch.randint(0, V, (B, T), generator=g, device="cuda"))
        return s
    s["u"] = torch.rand(B, T, generator=g, device="cuda")
    logits = 3.0 * _rn(g, B, T, V)
    s["target"] = torch.softmax(logits, -1)
    guess = logits + 0.4 * _rn(g, B, T, V)  # the draft knows the target about, not exactly
    if mode == "chain":
        if T == 1:
            s["draft"], s["tokens"] = torch.empty(B, 0, V, device="cuda"), torch.zeros(B, 1, dtype=torch.long, device="cuda")
            return s
        s["draft"] = torch.softmax(guess[:, :-1], -1)
        drawn = torch.multinomial(s["draft"].flatten(0, 1), 1, generator=g).view(B, T - 1)
        s["tokens"] = torch.cat([torch.zeros(B, 1, dtype=torch.long, device="cuda"), drawn], 1)
        return s
    # child r of a node carries the draft's r-th best token there
    best = guess.topk(min(8, V), -1).indices
    earlier = (s["parents"][:, :, None] == s["parents"][:, None, :]) & torch.ones(T, T, dtype=torch.bool, device="cuda").tril(-1)
    rank = earlier.sum(-1).clamp(max=best.shape[-1] - 1)
    s["tokens"] = best.gather(1, par[..., None].expand(-1, -1, best.shape[-1])).gather(2, rank[..., None]).squeeze(-1)
    return s


# ---------------------------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    return globals()[("_own_" if own else "_plain_") + c["kind"]](c, state)


def _own_rope(c, s):
    return s["rope"].rotate(s["x"], s["pos"], inverse=c["inverse"])


def _own_append(c, s):
    layer = s["cache"].layer(0)
    q = layer.append(s["k"], s["v"], s["start"], counts=s["counts"], q=s["q"], rope=s["rope"], positions=s["pos"])
    k, v = layer.read(s["start"], c["T"])
    return {"q": q, "k": k, "v": v}


def _own_read(c, s):
    k, v = s["cache"].layer(0).read(s["start"], c["n"])
    return {"k": k, "v": v}


def _own_attn(c, s):
    from sparse_transformers_b200 import tree_attention

    return tree_attention(s["q"], s["cache"].layer(0), s["length"], tree=s["sees"] if c["tree"] else None, counts=s["counts"])


def _own_verify(c, s):
    from sparse_transformers_b200 import verify_draft

    path, count, token = verify_draft(s["tokens"], s["target"], uniform=s.get("u"), parents=s["parents"] if c["mode"] != "chain" else None, draft=s.get("draft"), counts=s["counts"])
    return {"path": path, "count": count, "next": token}


def _turn(x, pos, w, f, layout, inverse=False):
    """x [..., heads, hd] in 32 bits turned by the angles pos * w (formed in 64 bits)."""
    rot = 2 * w.numel()
    a = pos.double()[..., None, None] * w
    cos, sin = (f * a.cos()).float(), ((-f if inverse else f) * a.sin()).float()
    x, rest = x[..., :rot], x[..., rot:]
    x0, x1 = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :rot // 2], x[..., rot // 2:])
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    y = torch.stack([y0, y1], -1).flatten(-2) if layout == "interleaved" else torch.cat([y0, y1], -1)
    return torch.cat([y, rest], -1)


def _plain_rope(c, s):
    return _turn(s["x"].float(), s["pos"], s["w"], s["f"], c["layout"], c["inverse"]).to(s["x"].dtype)


def _rows(c, s, n):
    """Indices (sequence, slot) of the n slots from each start on."""
    return torch.arange(c["B"], device="cuda")[:, None], s["start"][:, None] + torch.arange(n, device="cuda")


def _raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain_append(c, s):
    dt = s["q"].dtype
    q, k = (_turn(s[n].float(), s["pos"], s["w"], s["f"], c["layout"]) for n in ("q", "k"))
    used = torch.arange(c["T"], device="cuda") < s["counts"][:, None]
    b, slot = _rows(c, s, c["T"])
    back = []
    for x, cache, scale in ((k, s["kc"], s["ks"]), (s["v"].float(), s["vc"], s["vs"])):
        codes, top = _hold(x, c["store"], dt)
        raw = _raw(cache)
        raw[b, :, slot] = torch.where(used[..., None, None], _raw(codes), raw[b, :, slot])
        if scale is not None:
            scale[b, :, slot] = torch.where(used[..., None], top, scale[b, :, slot])
        back.append(_plain_rows(cache, scale, b, slot, dt))
    q = torch.where(used[..., None, None], q, torch.zeros_like(q)).to(dt)
    return {"q": q, "k": back[0], "v": back[1]}


def _plain_rows(cache, scale, b, slot, dt):
    codes = _raw(cache)[b, :, slot].view(cache.dtype)
    return _held(codes, None if scale is None else scale[b, :, slot]).transpose(1, 2).to(dt).contiguous()


def _plain_read(c, s):
    b, slot = _rows(c, s, c["n"])
    return {n: _plain_rows(s[n + "c"], s[n + "s"], b, slot, DTYPES[c["dtype"]]) for n in ("k", "v")}


def _plain_attn(c, s):
    rows, T, G = s["kc"].shape[2], c["T"], c["heads"] // c["kv"]
    k, v = _held(s["kc"], s["ks"]), _held(s["vc"], s["vs"])
    slot = torch.arange(rows, device="cuda")
    node = slot[None] - s["length"][:, None]                                              # [B,rows]
    bits = (s["sees"][:, :, None] >> node.clamp(0, T - 1)[:, None]) & 1                   # a chain's bits are a triangle
    sees = (node < 0)[:, None] | ((node >= 0) & (node < s["counts"][:, None]))[:, None] & (bits != 0)  # [B,T,rows]
    q = s["q"].float().unflatten(2, (c["kv"], G)).permute(0, 2, 3, 1, 4)                 # [B,kv,G,T,hd]
    score = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (G, T)) / math.sqrt(c["hd"])
    score = torch.where(sees[:, None, None], score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (G, T)) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                            # [B,T,heads,hd]
    used = torch.arange(T, device="cuda") < s["counts"][:, None]
    return torch.where(used[..., None, None], o, torch.zeros_like(o)).to(s["q"].dtype)


def _drawn(mass, u):
    """First index whose running sum is over u times the whole (64 bits); the last one of any weight where none is."""
    run_ = mass.cumsum(-1)
    whole = run_[..., -1:]
    over = run_ > u.double()[..., None] * whole
    last = mass.shape[-1] - 1 - (mass > 0).flip(-1).int().argmax(-1)
    j = torch.where(over.any(-1), over.int().argmax(-1), last)
    return torch.where((whole.squeeze(-1) > 0) & torch.isfinite(whole.squeeze(-1)), j, torch.full_like(j, -1))


def _plain_verify(c, s):
    B, T = c["B"], c["T"]
    node = torch.arange(T, device="cuda")
    used = node < s["counts"][:, None]
    one = torch.arange(B, device="cuda")
    if c["mode"] == "chain":
        p, q, x = s["target"], s["draft"], s["tokens"][:, 1:, None]
        took = s["u"][:, 1:].double() * q.gather(-1, x).squeeze(-1).double() < p[:, :-1].gather(-1, x).squeeze(-1).double()
        n = (took & used[:, 1:]).int().cumprod(1).sum(1)                                  # nodes taken behind the root
        refused = n + 1 < s["counts"]
        mass = p[one, n].double()
        if T > 1:
            rest = (mass - q[one, n.clamp(max=T - 2)].double()).clamp(min=0)
            mass = torch.where((refused & (rest.sum(-1) > 0))[:, None], rest, mass)
        return {"path": torch.where(node <= n[:, None], node, -1), "count": n + 1, "next": _drawn(mass, s["u"][:, 0])}
    draws = s["target"] if c["mode"] == "greedy" else _drawn(s["target"].double(), s["u"])  # [B,T]: the token behind each node
    par = s["parents"]
    hit = (node > 0) & used & (draws.gather(1, par.clamp(min=0)) == s["tokens"])
    twin = (par[:, :, None] == par[:, None, :]) & hit[:, None, :] & (node[None, :] < node[:, None])
    hit = (hit & ~twin.any(-1)) | (node == 0)
    sees = ((s["sees"][:, :, None] >> node) & 1) != 0                                     # [B,T,T]: ancestors and itself
    taken = (hit[:, None, :] | ~sees).all(-1) & used
    path = torch.where(taken, node, T).sort(-1).values
    path = torch.where(path < T, path, -1)
    count = taken.sum(-1)
    return {"path": path, "count": count, "next": draws[one, path[one, count - 1]]}


# ---------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    return globals()["_exact_" + c["kind"]](c, s)


def _exact_angles(c):
    """Angle per position of each pair and the factor, pair by pair."""
    rot, f, orig = c["rot"], c["factor"], c["orig"]
    got = []
    for i in range(rot // 2):
        base = c["theta"]
        if c["scaling"] == "ntk" and rot > 2:
            base *= math.pow(f, rot / (rot - 2.0))
        w = math.pow(base, -(2.0 * i) / rot)
        if c["scaling"] == "linear":
            w = w / f
        elif c["scaling"] == "llama3":
            length = 2 * math.pi / w  # of a turn, in tokens
            if length > orig:
                w = w / f
            elif length > orig / 4.0:
                share = (orig / length - 1.0) / 3.0
                w = (1 - share) * w / f + share * w
        elif c["scaling"] == "yarn":
            lo = max(0, math.floor(rot * math.log(orig / (32.0 * 2 * math.pi)) / (2 * math.log(base))))
            hi = min(rot - 1, math.ceil(rot * math.log(orig / (2 * math.pi)) / (2 * math.log(base))))
            share = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            w = share * (w / f) + (1 - share) * w
        got.append(w)
    return np.array(got), 0.1 * math.log(f) + 1.0 if c["scaling"] == "yarn" else 1.0


def _exact_turn(c, x, pos, inverse):
    """As multiplication of complex numbers."""
    w, f = _exact_angles(c)
    w = torch.from_numpy(w).to(x.device)
    n, half = c["rot"], c["rot"] // 2
    where = [(2 * i, 2 * i + 1) if c["layout"] == "interleaved" else (i, i + half) for i in range(half)]
    re, im = (torch.tensor([p[k] for p in where], device=x.device) for k in (0, 1))
    x = x.double()
    z = torch.complex(x[..., re], x[..., im])
    a = pos.double().reshape(*pos.shape, 1, 1) * w
    z = z * torch.polar(torch.full_like(a, f), -a if inverse else a)
    y = x.clone()
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _exact_rope(c, s):
    return _exact_turn(c, s["x"], s["pos"], c["inverse"])


def _exact_rows(x, store, dt):
    """What is read back of rows x (64 bits)."""
    if store == "same":
        return x.to(dt).double()
    top = x.abs().max(-1, keepdim=True).values
    step = top / MOST[store]
    y = torch.where(top > 0, x / step, torch.zeros_like(x))
    y = torch.floor(y + 0.5) if store == "int8" else y.float().to(torch.float8_e4m3fn).double()
    return y * step


def _exact_append(c, s):
    q, k = _exact_turn(c, s["q"], s["pos"], False), _exact_turn(c, s["k"], s["pos"], False)
    out = {"q": q, "k": [], "v": []}
    start, counts = _starts(c), _counts(c)
    for n, x, codes, scale in (("k", k, s["kc"], s["ks"]), ("v", s["v"].double(), s["vc"], s["vs"])):
        for b in range(c["B"]):
            old = codes[b, :, start[b]:start[b] + c["T"]].double()
            if scale is not None:
                old = old * scale[b, :, start[b]:start[b] + c["T"], None].double()
            new = _exact_rows(x[b], c["store"], DTYPES[c["dtype"]]).transpose(0, 1)
            old[:, :counts[b]] = new[:, :counts[b]]
            out[n].append(old)
        out[n] = torch.stack(out[n])
    for b in range(c["B"]):
        q[b, counts[b]:] = 0
    return out


def _exact_read(c, s):
    out = {}
    for n in ("k", "v"):
        codes, scale = s[n + "c"].double(), s[n + "s"]
        if scale is not None:
            codes = codes * scale.double()[..., None]
        out[n] = torch.stack([codes[b, :, b % 4:b % 4 + c["n"]] for b in range(c["B"])])
    return out


def _exact_attn(c, s):
    out = torch.zeros(c["B"], c["T"], c["heads"], c["hd"], dtype=torch.float64, device="cuda")
    G, sees = c["heads"] // c["kv"], s["sees"].cpu().numpy().view(np.uint64)
    for b, (l, n) in enumerate(zip(_lengths(c), _counts(c))):
        seen = torch.ones(n, l + n, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                seen[i, l + j] = bool((int(sees[b, i]) >> j) & 1)
        seen = seen.cuda()
        for h in range(c["kv"]):
            k, v = s["kc"][b, h, :l + n].double(), s["vc"][b, h, :l + n].double()
            if s["ks"] is not None:
                k, v = k * s["ks"][b, h, :l + n, None].double(), v * s["vs"][b, h, :l + n, None].double()
            for r in range(G):
                z = s["q"][b, :n, h * G + r].double() @ k.T * c["hd"] ** -0.5
                out[b, :n, h * G + r] = torch.softmax(z.masked_fill(~seen, -math.inf), -1) @ v
    return out


def _exact_verify(c, s):
    """Whole numbers only: none of them has a value between."""
    return None
