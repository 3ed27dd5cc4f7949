"""The work that a serving loop has an 8-bit key/value cache do, as a list of cases to be timed: new keys and values
quantised into the cache, attention over it, the attention weight that its keys have gathered, and eviction by that weight
(from a cache of either width).  Sizes are those of the benchmark configurations (triton_amd/configs.py) and of ordinary use
around them: one request and batches of ragged ones, one new token, a few drafted ones, chunks and whole prompts, caches from a
thousand keys to 131072.

A case is a dict of plain values: "op" names the operator, the rest its sizes.  An 8-bit cache holds e4m3 codes [batch, KV heads,
capacity, head_dim] and a float32 scale for each head and block of tokens.  `lengths` are the keys of each sequence, its new
tokens among them, and `counts` its new tokens; both lie on the GPU.  Where a case is ragged, the sequences of its batch have
from all down to about half of the stated tokens.
"""
import math

import torch

own = False

# query heads, KV heads, head_dim: the two benchmarked attention shapes, and two small generic ones
HEADS = {"llama": (32, 8, 128), "falcon": (71, 1, 64), "mha16": (16, 16, 64), "gqa8": (8, 2, 128)}
FLOOR = 2.0 ** -32          # the smallest scale: fp16's smallest number is 2^-24, e4m3's largest 1.75 * 2^8
MAX_BYTES = 9 << 26         # of a drawn case's cache: no more than the largest listed one's
MAX_PAIRS = 32 * 512 * 8448      # query heads x queries x keys of a drawn attention: no more than the listed chunk's


def listed():
    return [
        # one request's new token, a batch's new tokens on caches of many lengths, and a batch of prompts
        dict(name="append_token", op="append", heads="llama", batch=1, new=1, past=1024, block=64, ragged=False),
        dict(name="append_batch", op="append", heads="llama", batch=32, new=1, past=4096, block=64, ragged=True),
        dict(name="append_prompts", op="append", heads="llama", batch=4, new=2047, past=1000, block=64, ragged=True),
        # single tokens: one request on a short cache, a batch of ragged ones, one request on a long cache
        dict(name="attn_token", op="attn", heads="llama", batch=1, new=1, past=1024, block=64, ragged=False, causal=True),
        dict(name="attn_batch", op="attn", heads="llama", batch=32, new=1, past=8192, block=64, ragged=True, causal=True),
        dict(name="attn_long", op="attn", heads="llama", batch=1, new=1, past=131071, block=128, ragged=False, causal=True),
        # drafted tokens of many query heads on one KV head; a chunk of a prompt on the part before it
        dict(name="attn_drafts", op="attn", heads="falcon", batch=8, new=16, past=3001, block=64, ragged=True, causal=True),
        dict(name="attn_chunk", op="attn", heads="llama", batch=1, new=512, past=7936, block=64, ragged=False, causal=True),
        # with the weight that keys gather: a batch's decode step, and a whole prompt
        dict(name="weights_batch", op="weights", heads="llama", batch=16, new=1, past=4096, block=64, ragged=True, causal=True),
        dict(name="weights_prompt", op="weights", heads="llama", batch=1, new=1501, past=0, block=64, ragged=False, causal=True),
        # prompts cut down to a budget by their KeyFormer scores (one for each query head, as the drivers hold them in fp16),
        # and full 8-bit caches to half by the weight gathered
        dict(name="evict_prompts", op="evict", heads="llama", batch=4, past=4096, keep=1024, recent=256, bits=16, block=64, scores="query", ragged=True),
        dict(name="evict_cache8", op="evict", heads="llama", batch=16, past=8192, keep=4096, recent=64, bits=8, block=64, scores="kv", ragged=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "weights", "evict"])
    heads = rng.choice(["llama", "llama", "falcon", "mha16", "gqa8"])
    hq, hkv, d = HEADS[heads]
    block = rng.choice([32, 64, 64, 128])
    batch = _log_int(rng, 1, 32)
    room = MAX_BYTES // (2 * batch * hkv * d)          # tokens of each sequence
    if op == "append":
        new = rng.choice([1, _log_int(rng, 1, 2048)])
        return dict(op=op, heads=heads, batch=batch, new=min(new, max(1, 8192 // batch)), past=_log_int(rng, 1, min(8192, room // 2)), block=block, ragged=rng.random() < 0.5)
    if op == "evict":
        past = _log_int(rng, 64, min(16384, room // 2))
        keep = max(8, int(past * rng.uniform(0.2, 0.9)))
        return dict(op=op, heads=heads, batch=min(batch, 16), past=past, keep=keep, recent=int(keep * rng.uniform(0.0, 0.5)), bits=rng.choice([8, 16]),
                    block=block, scores=rng.choice(["query", "kv"]), ragged=rng.random() < 0.5)
    new = rng.choice([1, 1, _log_int(rng, 2, 32), _log_int(rng, 33, 1024)])
    past = _log_int(rng, 64, max(64, min(131072 if op == "attn" else 16384, room // 2, MAX_PAIRS // (batch * hq * new) - new)))
    while batch > 1 and batch * hq * new * (past + new) > MAX_PAIRS:
        batch -= 1
    return dict(op=op, heads=heads, batch=batch, new=new, past=past, block=block, ragged=rng.random() < 0.5, causal=rng.random() < 0.75)


# ------------------------------------------------------------------------------------------------ sizes
def _sizes(case):
    """(keys, new tokens) of each sequence, and the cache's capacity."""
    n, past, new = case["batch"], case["past"], case.get("new", 0)
    counts = [new - (b * new) // (2 * n) if case["ragged"] else new for b in range(n)]
    lengths = [(past - (b * past) // (2 * n) if case["ragged"] else past) + c for b, c in enumerate(counts)]
    return lengths, counts, past + new


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _keys(g, *shape):
    """Keys: a few channels are several times as large as the others."""
    loud = torch.where(torch.rand(shape[-1], generator=g, device="cuda") < 0.05, 6.0, 1.0)
    return (_randn(g, *shape) * loud).half()


def _values(g, *shape):
    """Values: tokens differ in size."""
    return (_randn(g, *shape) * torch.exp(0.5 * _randn(g, *shape[:-1], 1))).half()


def _need(amax):
    """The smallest power of two by which amax comes to no more than 448."""
    m, e = torch.frexp(amax.double())                        # amax = m 2^e, m in [1/2, 1); 448 = 0.875 2^9
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(m), e - 9 + (m > 0.875).to(e.dtype)), FLOOR).clamp(min=FLOOR).float()


def _by_block(x, block):
    """[batch, heads, tokens, ...] with the tokens in blocks, the last one filled up with zeros."""
    b, h, s = x.shape[:3]
    n = -(-s // block)
    full = torch.zeros((b, h, n * block) + x.shape[3:], dtype=x.dtype, device=x.device)
    full[:, :, :s] = x
    return full.view((b, h, n, block) + x.shape[3:])


def _quantised(x, block):
    """An 8-bit cache of x [batch, heads, tokens, head_dim]: codes and scales."""
    blocks = _by_block(x, block)
    scale = _need(blocks.abs().amax((3, 4)))
    codes = (blocks.float() / scale[..., None, None]).to(torch.float8_e4m3fn)
    return codes.flatten(2, 3)[:, :, :x.shape[2]].contiguous(), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    hq, hkv, d = HEADS[case["heads"]]
    n, (lengths, counts, cap), block = case["batch"], _sizes(case), case["block"]
    state = dict(case=case, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if case["op"] == "evict":
        k, v = _keys(g, n, hkv, cap, d), _values(g, n, hkv, cap, d)
        rows = hq if case["scores"] == "query" else hkv
        w = torch.exp(2.0 * _randn(g, n, rows, cap))
        state.update(weights=w.clamp(max=60000.0).half() if case["scores"] == "query" else w)
        keep = case["keep"]
        if case["bits"] == 8:
            (k, ks), (v, vs) = _quantised(k, block), _quantised(v, block)
            blocks = -(-keep // block)
            state.update(k_scale=ks, v_scale=vs, k_scale_out=torch.ones(n, hkv, blocks, device="cuda"), v_scale_out=torch.ones(n, hkv, blocks, device="cuda"))
        state.update(k=k, v=v, k_out=torch.zeros(n, hkv, keep, d, dtype=k.dtype, device="cuda"), v_out=torch.zeros(n, hkv, keep, d, dtype=k.dtype, device="cuda"),
                     weights_out=torch.zeros(n, rows, keep, dtype=state["weights"].dtype, device="cuda"),
                     kept=torch.full((n, hkv, keep), -1, dtype=torch.int32, device="cuda"), new_lengths=torch.zeros(n, dtype=torch.int32, device="cuda"))
        return state
    state["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    state["k8"], state["k_scale"] = _quantised(_keys(g, n, hkv, cap, d), block)
    state["v8"], state["v_scale"] = _quantised(_values(g, n, hkv, cap, d), block)
    new = case["new"]
    if case["op"] == "append":
        state.update(k=_keys(g, n, hkv, new, d), v=_values(g, n, hkv, new, d))
        return state
    # queries and outputs lie token by token, as the projections leave and take them
    state["q"] = _randn(g, n, new, hq, d).half().permute(0, 2, 1, 3)
    state["o"] = torch.zeros(n, new, hq, d, dtype=torch.float16, device="cuda").permute(0, 2, 1, 3)
    if case["op"] == "weights":
        state["weights"] = torch.rand(n, hkv, cap, generator=g, device="cuda") * 4.0
        state["weights_out"] = torch.zeros(n, hkv, cap, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _append_plain(x, codes, scale, lengths, counts, block):
    """New rows of x into codes and scale, in place, over the window of blocks that they touch."""
    n, h, m, d = x.shape
    s = codes.shape[2]
    first = (lengths - counts).long()
    blocks = min(-(-(m + block - 1) // block), scale.shape[2])
    base = (first // block).clamp(max=scale.shape[2] - blocks)                # the window's first block
    pos = base[:, None] * block + torch.arange(blocks * block, device=x.device)        # [n, window]
    row = pos - first[:, None]
    fresh = ((row >= 0) & (row < counts[:, None]))[:, None, :, None]
    at = pos.clamp(max=s - 1)[:, None, :, None].expand(n, h, -1, d)           # (places behind the cache's end stand for its last)
    new = x.gather(2, row.clamp(0, m - 1)[:, None, :, None].expand(n, h, -1, d)).float()
    old = codes.view(torch.uint8).gather(2, at)
    which = (base[:, None] + torch.arange(blocks, device=x.device))[:, None].expand(n, h, blocks)
    was = scale.gather(2, which)
    holds = (row < 0).view(n, 1, blocks, block).any(3)                        # rows before the new ones
    any_new = fresh.view(n, 1, blocks, block).any(3)
    need = _need((new.abs() * fresh).view(n, h, blocks, block * d).amax(3))
    now = torch.maximum(need, torch.where(holds, was, torch.full_like(was, FLOOR)))
    each = now.repeat_interleave(block, 2)[..., None]
    ratio = (was / now).repeat_interleave(block, 2)[..., None]
    before = ((row < 0) & any_new[:, 0].repeat_interleave(block, 1))[:, None, :, None]
    value = torch.where(fresh, new / each, old.view(torch.float8_e4m3fn).float() * ratio).to(torch.float8_e4m3fn).view(torch.uint8)
    final = torch.where(fresh | before, value, old)
    codes.view(torch.uint8).scatter_(2, at, final.gather(2, at - pos[:, :1, None, None]))
    scale.scatter_(2, which, torch.where(any_new, now, was))


def _attention_plain(state):
    """Probabilities [batch, KV heads, group, queries, keys], outputs, and which queries there are."""
    case, q = state["case"], state["q"]
    n, hq, m, d = q.shape
    hkv, s = state["k8"].shape[1:3]
    k, v = (state[c].float() * state[e].repeat_interleave(case["block"], 2)[:, :, :s, None] for c, e in (("k8", "k_scale"), ("v8", "v_scale")))
    t = (q.float().reshape(n, hkv, (hq // hkv) * m, d) @ k.transpose(2, 3)).view(n, hkv, hq // hkv, m, s) * d ** -0.5
    key, row = torch.arange(s, device=q.device), torch.arange(m, device=q.device)
    lengths, counts = state["lengths"][:, None, None], state["counts"][:, None, None]
    sees = (key < lengths) & (row[:, None] < counts)
    if case["causal"]:
        sees = sees & (key <= lengths - counts + row[:, None])
    sees = sees[:, None, None]
    t = t.masked_fill(~sees, -math.inf)
    top = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    o = (p.view(n, hkv, -1, s) @ v).view(n, hq, m, d)
    valid = (row < state["counts"][:, None])[:, None, :, None]
    return p, torch.where(valid, o.half(), state["o"])


def _evict_plain(state):
    case, w = state["case"], state["weights"]
    hkv, n = state["k"].shape[1:3]
    b, rows = w.shape[:2]
    keep, recent, block = case["keep"], case["recent"], case["block"]
    length = state["lengths"].long()[:, None, None]
    total = w.double().view(b, hkv, rows // hkv, n).sum(2).float()
    at = torch.arange(n, device=w.device)
    total = torch.where(at >= length, -math.inf, torch.where(at >= length - recent, math.inf, total))
    order = torch.sort(total, dim=2, descending=True, stable=True).indices[..., :keep]
    order = torch.where(order < length, order, n).sort(2).values                       # ascending; what is not there last
    there = order < length
    index = order.clamp(max=n - 1)
    out = {"kept": torch.where(there, order, -1).int(), "new_lengths": state["lengths"].clamp(max=keep)}
    by_row = index.repeat_interleave(rows // hkv, 1)
    out["weights"] = torch.where(there.repeat_interleave(rows // hkv, 1), w.gather(2, by_row), state["weights_out"])
    for name in ("k", "v"):
        x, to = state[name], state[name + "_out"]
        d = x.shape[3]
        take = index[..., None].expand(-1, -1, -1, d)
        if case["bits"] == 16:
            rows_ = x.gather(2, take)
            out[name] = torch.where(there[..., None], rows_, to)
        else:
            was = state[name + "_scale"].gather(2, index // block) * there
            now = _by_block(was, block).amax(3)
            rows_ = x.view(torch.uint8).gather(2, take).view(torch.float8_e4m3fn).float()
            rows_ = rows_ * (was / now.repeat_interleave(block, 2)[..., :keep])[..., None]
            rows_ = torch.where(there[..., None], rows_.to(torch.float8_e4m3fn).view(torch.uint8), to.view(torch.uint8))
            out[name] = rows_.view(torch.float8_e4m3fn)
            out[name + "_scale"] = torch.where(_by_block(there, block).any(3), now, state[name + "_scale_out"])
    return out


# ------------------------------------------------------------------------------------------------ one pass
def _own_module(state):
    """The module that a serving loop holds, made on the first pass."""
    from triton_amd import modules
    case = state["case"]
    if case["op"] == "append":
        return modules.get("append8", "cache", block=case["block"])
    if case["op"] == "evict":
        name = "evict8" if case["bits"] == 8 else "evict"
        return modules.get(name, "cache", keep=case["keep"], recent=case["recent"], **(dict(block=case["block"]) if case["bits"] == 8 else {}))
    return modules.get("attn8" if case["op"] == "attn" else "weights8", "cache", causal=case["causal"], block=case["block"])


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        if "module" not in state:
            module = state["module"] = _own_module(state)
            named = dict(K=state.get("k"), V=state.get("v"), K8=state.get("k8"), V8=state.get("v8"), K_scale=state.get("k_scale"), V_scale=state.get("v_scale"),
                         Q=state.get("q"), O=state.get("o"), weights=state.get("weights"), weights_out=state.get("weights_out"),
                         K_out=state.get("k_out"), V_out=state.get("v_out"), K_scale_out=state.get("k_scale_out"), V_scale_out=state.get("v_scale_out"),
                         kept=state.get("kept"), new_lengths=state.get("new_lengths"), lengths=state["lengths"], counts=state.get("counts"))
            state["args"] = [named[p] for p in module.TENSOR_PARAMS]
        state["module"].forward(*state["args"])
    if op == "append":
        if not own:
            for x, c, s in (("k", "k8", "k_scale"), ("v", "v8", "v_scale")):
                _append_plain(state[x], state[c], state[s], state["lengths"], state["counts"], case["block"])
        return dict(k8=state["k8"], v8=state["v8"], k_scale=state["k_scale"], v_scale=state["v_scale"])
    if op == "evict":
        if not own:
            return _evict_plain(state)
        out = dict(kept=state["kept"], new_lengths=state["new_lengths"], weights=state["weights_out"], k=state["k_out"], v=state["v_out"])
        if case["bits"] == 8:
            out.update(k_scale=state["k_scale_out"], v_scale=state["v_scale_out"])
        return out
    if own:
        return dict(o=state["o"], weights=state["weights_out"]) if op == "weights" else dict(o=state["o"])
    p, o = _attention_plain(state)
    if op == "attn":
        return dict(o=o)
    there = torch.arange(p.shape[-1], device=p.device) < state["lengths"][:, None, None]
    return dict(o=o, weights=torch.where(there, state["weights"] + p.sum((2, 3)), state["weights_out"]))


# ------------------------------------------------------------------------------------------------ least work
def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    lengths, counts, _ = _sizes(case)
    block = case["block"]
    if case["op"] == "append":
        # fp16 rows in, codes out, and a scale in and out for each block touched
        tokens = sum(counts)
        blocks = sum((n - 1) // block - (n - c) // block + 1 for n, c in zip(lengths, counts))
        return {"bytes": 2 * hkv * (tokens * d * 3 + blocks * 8), "flops": 2 * 2 * hkv * tokens * d}
    if case["op"] == "evict":
        rows, size = (hq, 2) if case["scores"] == "query" else (hkv, 4)
        kept = sum(min(n, case["keep"]) for n in lengths)
        width = case["bits"] // 8
        moved = 2 * kept * (2 * hkv * d * width + rows * size) + 4 * kept * hkv
        if case["bits"] == 8:
            moved += 2 * 4 * hkv * sum(-(-n // block) + -(-min(n, case["keep"]) // block) for n in lengths)
        return {"bytes": moved + sum(lengths) * rows * size, "flops": sum(lengths) * rows}
    blocks = sum(-(-n // block) for n in lengths)
    moved = 2 * hkv * (sum(lengths) * d + blocks * 4) + 2 * 2 * sum(counts) * hq * d
    # (a causal query sees the keys up to its own)
    pairs = sum(c * n - (c * (c - 1) // 2 if case["causal"] else 0) for n, c in zip(lengths, counts))
    if case["op"] == "weights":
        moved += 2 * 4 * hkv * sum(lengths)
    return {"bytes": moved, "flops": 4 * hq * d * pairs}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _e4m3(x):
    """The nearest number of 4 exponent and 3 mantissa bits (steps of 2^-9 below 2^-6), ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _least_scale(top):
    """For one largest magnitude (a float): the power of two."""
    scale = FLOOR
    while top > 448 * scale:
        scale *= 2
    return scale


def _append_exact(state, x, codes, scale, block):
    codes, scale = state[codes].float().double(), state[scale].double()
    top = state[x].double().abs().amax(3).cpu()
    for b, (n, c) in enumerate(zip(state["lengths"].tolist(), state["counts"].tolist())):
        for blk in range((n - c) // block, (n - 1) // block + 1):
            lo, hi = max(blk * block, n - c), min((blk + 1) * block, n)
            for h in range(codes.shape[1]):
                was = float(scale[b, h, blk]) if lo > blk * block else FLOOR
                now = max(was, _least_scale(float(top[b, h, lo - n + c:hi - n + c].max())))
                if lo > blk * block and now > was:
                    codes[b, h, blk * block:lo] = _e4m3(codes[b, h, blk * block:lo] * (was / now))
                codes[b, h, lo:hi] = _e4m3(state[x][b, h, lo - n + c:hi - n + c].double() / now)
                scale[b, h, blk] = now
    return codes, scale


def _attention_exact(state):
    case, q = state["case"], state["q"]
    hkv, block = state["k8"].shape[1], case["block"]
    group = q.shape[1] // hkv
    o = state["o"].double()
    weights = state["weights_out"].double() if "weights" in state else None
    for b, (n, c) in enumerate(zip(state["lengths"].tolist(), state["counts"].tolist())):
        key = torch.arange(n, device=q.device)
        hidden = key[None] > (n - c) + torch.arange(c, device=q.device)[:, None] if case["causal"] else None
        for h in range(hkv):
            k = state["k8"][b, h, :n].float().double() * state["k_scale"][b, h].double()[key // block][:, None]
            v = state["v8"][b, h, :n].float().double() * state["v_scale"][b, h].double()[key // block][:, None]
            gathered = 0.0
            for j in range(h * group, (h + 1) * group):
                t = torch.mm(q[b, j, :c].double(), k.t().contiguous()) / math.sqrt(q.shape[3])
                if hidden is not None:
                    t = t.masked_fill(hidden, -math.inf)
                p = torch.softmax(t, dim=1)
                o[b, j, :c] = torch.mm(p, v)
                gathered = gathered + p.sum(0)
            if weights is not None:
                weights[b, h, :n] = state["weights"][b, h, :n].double() + gathered
    return dict(o=o) if weights is None else dict(o=o, weights=weights)


def _evict_exact(state):
    case, w = state["case"], state["weights"].double()
    keep, block = case["keep"], case["block"]
    hkv = state["k"].shape[1]
    group = w.shape[1] // hkv
    out = dict(kept=state["kept"].clone(), new_lengths=torch.clamp(state["lengths"], max=keep), weights=state["weights_out"].double())
    for name in ("k", "v"):
        out[name] = state[name + "_out"].float().double()
        if case["bits"] == 8:
            out[name + "_scale"] = state[name + "_scale_out"].double()
    for b, n in enumerate(state["lengths"].tolist()):
        late = min(case["recent"], n)
        for h in range(hkv):
            total = w[b, h * group:(h + 1) * group, :n].sum(0).float()
            # (numbering the ties from the front: the earlier of two equal ones is the larger)
            early = sorted(range(n - late), key=(lambda s: lambda i: (-s[i], i))(total.tolist()))[:max(0, min(n, keep) - late)]
            index = torch.tensor(sorted(early) + list(range(n - late, n)), device=w.device)
            m = len(index)
            out["kept"][b, h, :m] = index.int()
            out["weights"][b, h * group:(h + 1) * group, :m] = w[b, h * group:(h + 1) * group][:, index]
            for name in ("k", "v"):
                rows = state[name][b, h][index].double() if case["bits"] == 16 else state[name][b, h].float()[index].double()
                if case["bits"] == 8:
                    was = state[name + "_scale"][b, h].double()[index // block]
                    for i in range(0, m, block):
                        now = was[i:i + block].max()
                        out[name + "_scale"][b, h, i // block] = now
                        rows[i:i + block] = _e4m3(rows[i:i + block] * (was[i:i + block] / now)[:, None])
                out[name][b, h, :m] = rows
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        if case["batch"] * HEADS[case["heads"]][1] * (case["new"] // case["block"] + 2) > 20000:
            return None                                      # (block by block in Python)
        (k8, ks), (v8, vs) = _append_exact(state, "k", "k8", "k_scale", case["block"]), _append_exact(state, "v", "v8", "v_scale", case["block"])
        return dict(k8=k8, v8=v8, k_scale=ks, v_scale=vs)
    if case["op"] == "evict":
        if case["batch"] * HEADS[case["heads"]][1] * case["past"] > 1 << 21:
            return None                                      # (sorted in Python)
        return _evict_exact(state)
    return _attention_exact(state)
