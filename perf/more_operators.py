"""The work that a serving loop has an fp16 key/value cache do whose sequences have lengths of their own, as a list of cases to be timed:
new queries and keys normalised by head, rotated by their positions and put into the cache with the values ("rope"); attention over a prefix
that all sequences of a batch share and over each one's own keys ("prefix"); attention over those blocks of a long cache that a cheap score
selects for each query ("sparse", with the blocks' bounds brought up to date).  Sizes are those of the benchmark configurations
(triton_amd/configs.py) and of ordinary use around them.

A case is a dict of plain values: "op" names the operator, the rest its sizes.  `lengths` are the keys that each sequence has of its own, its new tokens
among them, and `counts` its new tokens; both lie on the GPU.  Where a case is ragged, the sequences of its batch have from all down to about half of the
stated tokens.  Every value that an operator delivers in fp16 is rounded once, from 32 bits.
"""
import math

import torch

own = False

# query heads, KV heads, head_dim: the two benchmarked attention shapes, and two small generic ones
HEADS = {"llama": (32, 8, 128), "falcon": (71, 1, 64), "mha16": (16, 16, 64), "gqa8": (8, 2, 128)}
BASE = 500000.0             # of the rotations' frequencies, BASE^(-2 i / rotated dimensions)
EPS = 1e-6                  # of the norms


def listed():
    return [
        # one request's new token; a batch's new tokens, normalised by head; prompts, likewise, on caches that hold something; images and video among the
        # tokens: positions of three axes, half of each head rotated
        dict(name="rope_token", op="rope", heads="llama", batch=1, new=1, past=1024, ragged=False, norm=False, interleaved=False, rotated=128, axes=1),
        dict(name="rope_batch", op="rope", heads="llama", batch=48, new=1, past=100000, ragged=True, norm=True, interleaved=False, rotated=128, axes=1),
        dict(name="rope_prompts", op="rope", heads="llama", batch=4, new=2047, past=1000, ragged=True, norm=True, interleaved=False, rotated=128, axes=1),
        dict(name="rope_video", op="rope", heads="mha16", batch=2, new=8190, past=30, ragged=False, norm=False, interleaved=True, rotated=32, axes=3),
        # a few answers sampled from one short prompt; many from a long one, each some way on; drafted tokens of many query heads on one KV head; several
        # requests' prompts behind one long instruction
        dict(name="prefix_few", op="prefix", heads="llama", batch=4, new=1, past=60, prefix=1000, ragged=False),
        dict(name="prefix_samples", op="prefix", heads="llama", batch=32, new=1, past=700, prefix=8192, ragged=True),
        dict(name="prefix_drafts", op="prefix", heads="falcon", batch=16, new=5, past=301, prefix=16001, ragged=True),
        dict(name="prefix_prompts", op="prefix", heads="llama", batch=4, new=500, past=0, prefix=4000, ragged=True),
        # single tokens: one request on a medium cache, a batch of ragged ones, one on a long cache; a chunk of a long prompt
        dict(name="sparse_token", op="sparse", heads="llama", batch=1, new=1, past=8191, block=64, top=32, sink=1, recent=2, ragged=False),
        dict(name="sparse_batch", op="sparse", heads="llama", batch=16, new=1, past=30000, block=64, top=40, sink=1, recent=4, ragged=True),
        dict(name="sparse_long", op="sparse", heads="gqa8", batch=1, new=1, past=131071, block=32, top=128, sink=2, recent=8, ragged=False),
        dict(name="sparse_chunk", op="sparse", heads="llama", batch=1, new=256, past=32500, block=64, top=32, sink=1, recent=4, ragged=False),
    ]


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 5e14


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _drawn(rng):
    op = rng.choice(["rope", "prefix", "prefix", "sparse", "sparse"])
    case = dict(op=op, heads=rng.choice(["llama", "llama", "falcon", "mha16", "gqa8"]), ragged=rng.random() < 0.5)
    d = HEADS[case["heads"]][2]
    if op == "rope":
        axes = rng.choice([1, 1, 1, 2, 3])
        return dict(case, batch=_log_int(rng, 1, 64), new=rng.choice([1, _log_int(rng, 1, 8192)]), past=_log_int(rng, 1, 131072), norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.3, rotated=rng.choice([d, d, d // 2, 32]), axes=axes)
    new = rng.choice([1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 512)])
    if op == "prefix":
        return dict(case, batch=_log_int(rng, 1, 64), new=new, past=_log_int(rng, 1, 4096) - 1, prefix=_log_int(rng, 64, 65536))
    top = _log_int(rng, 4, 128)
    recent = _log_int(rng, 1, max(1, top // 4))
    return dict(case, batch=_log_int(rng, 1, 32), new=new, past=_log_int(rng, 256, 131072), block=rng.choice([32, 64, 64, 128]), top=top, sink=rng.randint(0, min(2, top - recent)),
                recent=recent)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("rope", "prefix", "sparse")}
    while True:
        case = _drawn(rng)
        hq, hkv, d = HEADS[case["heads"]]
        cache = 4 * case["batch"] * hkv * d * (case["past"] + case["new"])
        if _cost(case) <= most[case["op"]] and cache <= 1 << 31:
            return case


# ------------------------------------------------------------------------------------------------ sizes
def _sizes(case):
    """(own keys, new tokens) of each sequence, and the cache's capacity."""
    n, past, new = case["batch"], case["past"], case["new"]
    counts = [new - (b * new) // (2 * n) if case["ragged"] else new for b in range(n)]
    lengths = [(past - (b * past) // (2 * n) if case["ragged"] else past) + c for b, c in enumerate(counts)]
    return lengths, counts, past + new


def _sections(case):
    """How many pairs each axis has; the first one, time, as many as are left over."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    each = 3 * pairs // (4 * axes) if axes > 1 else 0
    return [pairs - (axes - 1) * each] + [each] * (axes - 1)


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _loud(g, d):
    """A few channels of the keys are several times as large as the others."""
    return torch.where(torch.rand(d, generator=g, device="cuda") < 0.05, 4.0, 1.0)


def _values(g, *shape):
    """Values: tokens differ in size."""
    return (_randn(g, *shape) * torch.exp(0.5 * _randn(g, *shape[:-1], 1))).half()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    hq, hkv, d = HEADS[case["heads"]]
    n, new, (lengths, counts, cap) = case["batch"], case["new"], _sizes(case)
    state = dict(case=case, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    if case["op"] == "rope":
        # queries, keys and values lie token by token beside each other, as the projection leaves them
        qkv = _randn(g, n, new, hq + 2 * hkv, d).half().permute(0, 2, 1, 3)
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], q_out=torch.zeros(n, new, hq, d, dtype=torch.float16, device="cuda").permute(0, 2, 1, 3))
        state.update(k_cache=torch.zeros(n, hkv, cap, d, dtype=torch.float16, device="cuda"), v_cache=torch.zeros(n, hkv, cap, d, dtype=torch.float16, device="cuda"))
        pairs = case["rotated"] // 2
        state["inv_freq"] = BASE ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
        state["gamma_q"], state["gamma_k"] = ((1 + 0.1 * _randn(g, d)).half() if case["norm"] else None for _ in range(2))
        # (which axis a pair turns with: of the plain form alone)
        state["axis"] = torch.tensor([a for a, many in enumerate(_sections(case)) for _ in range(many)], device="cuda")
        state["positions"] = None
        if case["axes"] > 1:
            # frames of 24 x 24 or so behind the keys that are there, a new first frame for each set of inputs
            t = torch.arange(new, device="cuda")[None] + torch.randint(0, 500, (n, 1), generator=g, device="cuda")
            at = [t // 576 + (state["lengths"] - state["counts"])[:, None], t % 576 // 24, t % 24]
            state["positions"] = torch.stack(at[:case["axes"]]).int()
        return state
    loud = _loud(g, d)
    # queries and outputs lie token by token, as the projections leave and take them
    state["o"] = torch.zeros(n, new, hq, d, dtype=torch.float16, device="cuda").permute(0, 2, 1, 3)
    state["v"] = _values(g, n, hkv, cap, d)
    if case["op"] == "prefix":
        state["q"] = _randn(g, n, new, hq, d).half().permute(0, 2, 1, 3)
        state["k"] = (_randn(g, n, hkv, cap, d) * loud).half()
        state.update(k_prefix=(_randn(g, hkv, case["prefix"], d) * loud).half(), v_prefix=_values(g, hkv, case["prefix"], d))
        return state
    # keys of a hundred tokens or so are alike, and a query asks for some of these subjects
    subjects = _randn(g, n, hkv, -(-cap // 100), d)
    which = ((torch.arange(cap, device="cuda") + 37) // 100).clamp(max=subjects.shape[2] - 1)
    state["k"] = ((0.8 * _randn(g, n, hkv, cap, d) + 0.6 * subjects[:, :, which]) * loud).half()
    asked = torch.randint(0, subjects.shape[2], (n, hkv, new), generator=g, device="cuda")[..., None].expand(-1, -1, -1, d)
    q = _randn(g, n, new, hkv, hq // hkv, d) + 0.5 * subjects.gather(2, asked).permute(0, 2, 1, 3)[:, :, :, None]
    state["q"] = q.flatten(2, 3).half().permute(0, 2, 1, 3)
    # the bounds of the keys that were there before
    block = case["block"]
    old = (state["lengths"] - state["counts"])[:, None, None, None]
    there = torch.arange(cap, device="cuda")[None, None, :, None] < old
    state["bounds"] = torch.stack([_by_block(torch.where(there, state["k"], fill), block, fill).amin(3) if fill > 0 else
                                   _by_block(torch.where(there, state["k"], fill), block, fill).amax(3) for fill in (65504.0, -65504.0)], 3).half()
    state["selected"] = torch.full((n, hkv, new, case["top"]), -1, dtype=torch.int32, device="cuda")
    return state


def _by_block(x, block, fill):
    """[batch, heads, tokens, ...] with the tokens in blocks, the last one filled up."""
    b, h, s = x.shape[:3]
    n = -(-s // block)
    full = torch.full((b, h, n * block) + x.shape[3:], fill, dtype=x.dtype, device=x.device)
    full[:, :, :s] = x
    return full.view((b, h, n, block) + x.shape[3:])


# ------------------------------------------------------------------------------------------------ plain forms
def _rope_plain(state):
    case, lengths, counts = state["case"], state["lengths"].long(), state["counts"].long()
    n, _, m, d = state["q"].shape
    row = torch.arange(m, device=lengths.device)
    to = (lengths - counts)[:, None] + row                                     # [n, m]: where new tokens go
    fresh = row < counts[:, None]
    at = state["positions"] if state["positions"] is not None else to[None]
    angle = at.double()[state["axis"]].permute(1, 2, 0) * state["inv_freq"]              # [n, m, pairs], in 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, gamma):
        x = x.float()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.float()
        pairs = case["rotated"] // 2
        if case["interleaved"]:
            a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
            first = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :pairs], x[..., pairs:2 * pairs]
            first = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([first, x[..., 2 * pairs:]], -1).half()

    q_out = torch.where(fresh[:, None, :, None], turned(state["q"], state["gamma_q"]), state["q_out"])
    out = [q_out]
    for x, cache in ((turned(state["k"], state["gamma_k"]), state["k_cache"]), (state["v"], state["v_cache"])):
        cap = cache.shape[2]
        # (rows that are not there write what the cache's first rows before the new ones hold)
        old = to.clamp(max=cap - 1)[:, None, :, None].expand(-1, x.shape[1], -1, d)
        cache.scatter_(2, old, torch.where(fresh[:, None, :, None], x, cache.gather(2, old)))
        out.append(cache)
    return out


def _prefix_plain(state):
    q, k, v, kp, vp = (state[c].float() for c in ("q", "k", "v", "k_prefix", "v_prefix"))
    n, hq, m, d = q.shape
    hkv, s = k.shape[1:3]
    p = kp.shape[1]
    q = q.reshape(n, hkv, (hq // hkv) * m, d)
    t = torch.empty(n, hkv, hq // hkv, m, p + s, device=q.device)
    t[..., :p] = (q.transpose(0, 1).reshape(hkv, -1, d) @ kp.transpose(1, 2)).view(hkv, n, -1, m, p).transpose(0, 1) * d ** -0.5
    t[..., p:] = (q @ k.transpose(2, 3)).view(n, hkv, -1, m, s) * d ** -0.5
    key, row = torch.arange(s, device=q.device), torch.arange(m, device=q.device)
    lengths, counts = state["lengths"][:, None, None], state["counts"][:, None, None]
    hidden = key > lengths - counts + row[:, None]                             # [n, m, s]
    t[..., p:].masked_fill_(hidden[:, None, None], -math.inf)
    e = torch.exp(t - t.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    o = (e[..., :p].transpose(0, 1).reshape(hkv, -1, p) @ vp).view(hkv, n, hq // hkv, m, d).transpose(0, 1) + (e[..., p:].reshape(n, hkv, -1, s) @ v).view(n, hkv, -1, m, d)
    fresh = (row < state["counts"][:, None])[:, None, :, None]
    return torch.where(fresh, o.reshape(n, hq, m, d).half(), state["o"])


def _bounds_plain(state):
    """The bounds of all keys: those of blocks that the new ones do not touch are what they were."""
    block, k = state["case"]["block"], state["k"]
    s = k.shape[2]
    key = torch.arange(s, device=k.device)[None, None, :, None]
    there = key < state["lengths"][:, None, None, None]
    lo = _by_block(torch.where(there, k, math.inf), block, math.inf).amin(3)
    hi = _by_block(torch.where(there, k, -math.inf), block, -math.inf).amax(3)
    nth = torch.arange(lo.shape[2], device=k.device)
    length, count = state["lengths"][:, None], state["counts"][:, None]
    touched = (count > 0) & (nth >= (length - count) // block) & (nth * block < length)
    state["bounds"].copy_(torch.where(touched[:, None, :, None, None], torch.stack([lo, hi], 3), state["bounds"]))
    return state["bounds"]


def _sparse_plain(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    n, hq, m, d = q.shape
    hkv, s = k.shape[1:3]
    g, block, top = hq // hkv, case["block"], case["top"]
    bounds = _bounds_plain(state)
    nb = bounds.shape[2]
    # the most that a key within the bounds can score, in 64 bits; of a KV head's query heads the largest, rounded to 32
    qq = q.double().reshape(n, hkv, g * m, d)
    best = qq.clamp(min=0) @ bounds[:, :, :, 1].double().transpose(2, 3).contiguous() + qq.clamp(max=0) @ bounds[:, :, :, 0].double().transpose(2, 3).contiguous()
    best = best.view(n, hkv, g, m, nb).amax(2).float()                         # [n, hkv, m, blocks]
    row, nth = torch.arange(m, device=q.device), torch.arange(nb, device=q.device)
    last = (state["lengths"] - state["counts"])[:, None] + row                  # [n, m]: the last key that a query sees
    ends = (last // block)[:, None, :, None]
    best = torch.where((nth < case["sink"]) | (nth > ends - case["recent"]), math.inf, best)
    best = torch.where(nth > ends, -math.inf, best)
    order = torch.sort(best, dim=3, descending=True, stable=True).indices[..., :top]
    order = torch.where(order <= ends, order, nb).sort(3).values                # ascending; what is not there last
    chosen = torch.where(order < nb, order, -1).int()
    if top > nb:
        chosen = torch.cat([chosen, chosen.new_full((n, hkv, m, top - nb), -1)], 3)
    fresh = row < state["counts"][:, None]
    selected = torch.where(fresh[:, None, :, None], chosen, state["selected"])
    # keys and values of each query
    keys = (chosen.long()[..., None] * block + torch.arange(block, device=q.device)).flatten(3)        # [n, hkv, m, top * block]
    sees = (keys >= 0) & (keys <= last[:, None, :, None]) & chosen.ge(0).repeat_interleave(block, 3)
    take = keys.clamp(0, s - 1).flatten(2)[..., None].expand(-1, -1, -1, d)
    kk, vv = (x.gather(2, take).view(n, hkv, m, -1, d).float() for x in (k, v))
    t = (q.float().reshape(n, hkv, g, m, d).transpose(2, 3) @ kk.transpose(3, 4)) * d ** -0.5           # [n, hkv, m, g, keys]
    t = t.masked_fill(~sees[:, :, :, None], -math.inf)
    e = torch.exp(t - t.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)) @ vv
    o = o.transpose(2, 3).reshape(n, hq, m, d).half()
    return [bounds, selected, torch.where(fresh[:, None, :, None], o, state["o"])]


# ------------------------------------------------------------------------------------------------ one pass
def _own_modules(state):
    """The modules that a serving loop holds, made on the first pass, with their tensors in order."""
    from triton_amd import modules
    case = state["case"]
    if case["op"] == "rope":
        made = [modules.get("rope", "cache", norm=case["norm"], eps=EPS, interleaved=case["interleaved"], sections=_sections(case))]
    elif case["op"] == "prefix":
        made = [modules.get("prefix", "cache")]
    else:
        made = [modules.get("bounds", "cache", block=case["block"]),
                modules.get("sparse", "cache", block=case["block"], top=case["top"], sink=case["sink"], recent=case["recent"])]
    named = dict(Q=state.get("q"), K=state.get("k"), V=state.get("v"), O=state.get("o"), Q_out=state.get("q_out"), K_cache=state.get("k_cache"),
                 V_cache=state.get("v_cache"), K_prefix=state.get("k_prefix"), V_prefix=state.get("v_prefix"), inv_freq=state.get("inv_freq"),
                 gamma_q=state.get("gamma_q"), gamma_k=state.get("gamma_k"), positions=state.get("positions"), bounds=state.get("bounds"),
                 selected=state.get("selected"), lengths=state["lengths"], counts=state["counts"])
    return [(m, [named[p] for p in m.TENSOR_PARAMS]) for m in made]


def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "rope":
            return dict(zip(("q_out", "k_cache", "v_cache"), _rope_plain(state)))
        return dict(o=_prefix_plain(state)) if op == "prefix" else dict(zip(("bounds", "selected", "o"), _sparse_plain(state)))
    if "modules" not in state:
        state["modules"] = _own_modules(state)
    for module, tensors in state["modules"]:
        module.forward(*tensors)
    return {name: state[name] for name in {"rope": ("q_out", "k_cache", "v_cache"), "prefix": ("o",), "sparse": ("bounds", "selected", "o")}[op]}


# ------------------------------------------------------------------------------------------------ least work
def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    lengths, counts, _ = _sizes(case)
    tokens = sum(counts)
    if case["op"] == "rope":
        positions = 4 * case["axes"] * tokens if case["axes"] > 1 else 0
        return {"bytes": 2 * 2 * tokens * (hq + 2 * hkv) * d + positions, "flops": tokens * (hq + hkv) * (3 * case["rotated"] + (4 * d if case["norm"] else 0))}
    moved = 2 * 2 * tokens * hq * d                                             # queries and outputs
    if case["op"] == "prefix":
        # (a query sees the prefix and its own keys up to itself)
        pairs = sum(c * (case["prefix"] + n) - c * (c - 1) // 2 for n, c in zip(lengths, counts))
        return {"bytes": moved + 2 * 2 * hkv * d * (case["prefix"] + sum(lengths)), "flops": 4 * hq * d * pairs}
    block, top = case["block"], case["top"]
    flops = 0
    for n, c in zip(lengths, counts):
        blocks, pairs, keys = 0, 0, 0                                           # scored, attended to, and those read for the latter
        for p in range(n - c, n):
            seen = p // block + 1
            mine = (min(top, seen) - 1) * block + p % block + 1
            blocks, pairs, keys = blocks + seen, pairs + mine, keys + mine
        flops += 4 * hq * d * (blocks + pairs)
        touched = (n - 1) // block - (n - c) // block + 1
        moved += hkv * (2 * 2 * d * min(n, keys) + 2 * 2 * d * ((n - 1) // block + 1 + touched) + 4 * c * top)
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _rope_exact(state):
    case = state["case"]
    pairs, start = case["rotated"] // 2, [0]
    for s in _sections(case):
        start.append(start[-1] + s)
    out = [state["q_out"].double(), state["k_cache"].double(), state["v_cache"].double()]
    for b, (n, c) in enumerate(zip(state["lengths"].tolist(), state["counts"].tolist())):
        angle = torch.empty(c, pairs, dtype=torch.float64, device="cuda")
        for a in range(case["axes"]):
            at = torch.arange(n - c, n, device="cuda") if state["positions"] is None else state["positions"][a, b, :c]
            angle[:, start[a]:start[a + 1]] = at.double()[:, None] * state["inv_freq"][start[a]:start[a + 1]]
        turn = torch.polar(torch.ones_like(angle), angle)
        for i, name in enumerate(("q", "k")):
            x = state[name][b, :, :c].double()
            if case["norm"]:
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * state["gamma_" + name].double()
            first = list(range(0, 2 * pairs, 2)) if case["interleaved"] else list(range(pairs))
            second = [j + 1 for j in first] if case["interleaved"] else [j + pairs for j in first]
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            if name == "q":
                out[0][b, :, :c] = x
            else:
                out[1][b, :, n - c:n] = x
        out[2][b, :, n - c:n] = state["v"][b, :, :c].double()
    return out


def _prefix_exact(state):
    q, o = state["q"], state["o"].double()
    group = q.shape[1] // state["k"].shape[1]
    for b, (n, c) in enumerate(zip(state["lengths"].tolist(), state["counts"].tolist())):
        for h in range(q.shape[1]):
            k = torch.cat([state["k_prefix"][h // group], state["k"][b, h // group, :n]]).double()
            v = torch.cat([state["v_prefix"][h // group], state["v"][b, h // group, :n]]).double()
            t = torch.mm(q[b, h, :c].double(), k.t().contiguous()) / math.sqrt(q.shape[3])
            late = torch.arange(len(k), device="cuda")[None] > len(k) - c + torch.arange(c, device="cuda")[:, None]
            o[b, h, :c] = torch.mm(torch.softmax(t.masked_fill(late, -math.inf), dim=1), v)
    return o


def _sparse_exact(state):
    case, q, k = state["case"], state["q"], state["k"]
    block, top, group = case["block"], case["top"], q.shape[1] // k.shape[1]
    bounds, selected, o = state["bounds"].double(), state["selected"].clone(), state["o"].double()
    for b, (n, c) in enumerate(zip(state["lengths"].tolist(), state["counts"].tolist())):
        for blk in range((n - c) // block, (n - 1) // block + 1):
            rows = k[b, :, blk * block:min(n, (blk + 1) * block)].double()
            bounds[b, :, blk, 0], bounds[b, :, blk, 1] = rows.min(1).values, rows.max(1).values
        nb = (n - 1) // block + 1
        for h in range(k.shape[1]):
            mine = q[b, h * group:(h + 1) * group, :c].double()
            # a channel's larger product, of its lower and of its upper bound
            score = torch.full((c, nb), -math.inf, dtype=torch.float64, device="cuda")
            for j in range(group):
                centre, half = (bounds[b, h, :nb, 0] + bounds[b, h, :nb, 1]) / 2, (bounds[b, h, :nb, 1] - bounds[b, h, :nb, 0]) / 2
                score = torch.maximum(score, torch.mm(mine[j], centre.t().contiguous()) + torch.mm(mine[j].abs(), half.t().contiguous()))
            score = score.float().tolist()
            see = torch.zeros(c, n, dtype=torch.bool)
            for i in range(c):
                ends = (n - c + i) // block
                forced = [x for x in range(ends + 1) if x < case["sink"] or x > ends - case["recent"]][:top]
                others = sorted((x for x in range(case["sink"], ends - case["recent"] + 1)), key=lambda x: (-score[i][x], x))
                blocks = sorted(forced + others[:max(0, top - len(forced))])
                selected[b, h, i] = torch.tensor(blocks + [-1] * (top - len(blocks)), dtype=torch.int32)
                for x in blocks:
                    see[i, x * block:min((x + 1) * block, n - c + i + 1)] = True
            see = see.cuda()
            kk, vv = k[b, h, :n].double(), state["v"][b, h, :n].double()
            for j in range(group):
                t = torch.mm(mine[j], kk.t().contiguous()) / math.sqrt(q.shape[3])
                o[b, h * group + j, :c] = torch.mm(torch.softmax(t.masked_fill(~see, -math.inf), dim=1), vv)
    return [bounds, selected, o]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope":
        return dict(zip(("q_out", "k_cache", "v_cache"), _rope_exact(state)))
    if case["op"] == "prefix":
        return dict(o=_prefix_exact(state))
    hkv = HEADS[case["heads"]][1]
    if case["batch"] * hkv * case["new"] * (case["past"] // case["block"] + 10) > 1 << 22:
        return None                                          # (selected in Python)
    return dict(zip(("bounds", "selected", "o"), _sparse_exact(state)))
