"""The attention layer's serving operators, their plain forms and the cases they are measured on.

``qk_norm_rope`` norms and rotates queries and keys for the dense attention, ``rope_append`` does the same for a ragged
batch of new tokens and puts its keys and values into the pages of the decode cache, ``attn_paged`` attends with those
tokens over that cache.  With ``own`` false ``run`` computes them from elementary torch operations in 32 bits (angles in
64), with ``own`` true it calls the framework.
"""

import math
import random
import sys

import torch

own = False

PAGE = 64          # rows of a page of the decode cache
HEAD = 128         # its head dimension
EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the first chunk of one prompt, nothing cached: causal self-attention, the tensor cores' case
        _attend("attend first chunk bf16", "bf16", 32, 8, "even", 1, 4096, 0),
        # a later chunk of a long document: the largest call, every row sees most of a 32048-row cache
        _attend("attend long cache bf16", "bf16", 32, 8, "even", 1, 2048, 30000),
        # a serving step: one prompt chunk beside fifteen sequences that decode one token each
        _attend("attend mixed step f16", "f16", 32, 8, "mixed", 16, 499, 7600),
        # a few drafted tokens of one short sequence to verify: latency
        _attend("attend verify small bf16", "bf16", 32, 8, "even", 1, 5, 1000),
        # drafted tokens of a batch of long sequences with ragged lengths, group of 5 heads: the cache's bandwidth
        _attend("attend verify batch bf16", "bf16", 40, 8, "ragged", 32, 7, 16001),
        # one token of one sequence: the smallest append, latency
        _append("append one token bf16", "bf16", 32, 8, "even", 1, 1, 777, HEAD, False, True),
        # a decode step of a batch, no norms
        _append("append decode batch f16", "f16", 32, 8, "ragged1", 64, 1, 32000, HEAD, False, False),
        # a prompt chunk, with norms
        _append("append chunk bf16", "bf16", 32, 8, "even", 2, 8192, 0, HEAD, False, True),
        # ragged chunks, neighbouring pairs rotated, half of the head, far positions
        _append("append ragged far f16", "f16", 24, 3, "ragged", 9, 301, 900000, 64, True, True),
        # the dense attention's benchmark shape, head-major outputs
        _rotate("rotate 8x4096 bf16", "bf16", 8, 4096, 32, 32, 128, 128, False, True),
        # 32-bit path of the dense attention
        _rotate("rotate 1x256 f32", "f32", 1, 256, 4, 4, 64, 64, False, True),
        # odd length, grouped heads, a head of 96 with a third of it rotated in neighbouring pairs, no norms
        _rotate("rotate odd f16", "f16", 3, 1021, 12, 4, 96, 32, True, False),
    ]


def _attend(name, dtype, hq, hkv, kind, batch, tokens, cached, mix=1):
    return {"name": name, "op": "attn_paged", "dtype": dtype, "hq": hq, "hkv": hkv, "kind": kind, "batch": batch,
            "tokens": tokens, "cached": cached, "mix": mix}


def _append(name, dtype, hq, hkv, kind, batch, tokens, cached, rot, neighbours, norm, mix=1):
    return {"name": name, "op": "rope_append", "dtype": dtype, "hq": hq, "hkv": hkv, "kind": kind, "batch": batch,
            "tokens": tokens, "cached": cached, "rot": rot, "neighbours": neighbours, "norm": norm, "mix": mix}


def _rotate(name, dtype, batch, length, hq, hkv, dim, rot, neighbours, norm):
    return {"name": name, "op": "qk_norm_rope", "dtype": dtype, "batch": batch, "length": length, "hq": hq, "hkv": hkv,
            "dim": dim, "rot": rot, "neighbours": neighbours, "norm": norm}


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["attn_paged", "attn_paged", "rope_append", "qk_norm_rope"])
    if op == "qk_norm_rope":
        dtype = rng.choice(["bf16", "f16", "f32"])
        dim = 16 * rng.randint(2, 16)
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 3, 4, 8])
        batch = _spread(rng, 1, 8)
        room = (1 << 28) // (SIZES[dtype] * dim * (hq + hkv) * batch)   # half of the largest listed case's bytes
        length = _spread(rng, 1, max(1, min(8192, room)))
        case = _rotate("", dtype, batch, length, hq, hkv, dim, 16 * rng.randint(1, dim // 16), rng.random() < 0.5,
                       rng.random() < 0.6)
    elif op == "rope_append":
        kind = rng.choice(["even", "ragged", "ragged1"])
        hkv = rng.randint(1, 8)
        batch = _spread(rng, 1, 64)
        tokens = 1 if kind == "ragged1" else _spread(rng, 1, 8192 // batch)
        case = _append("", rng.choice(["bf16", "f16"]), hkv * rng.choice([1, 2, 3, 4, 5, 8]), hkv, kind, batch, tokens,
                       rng.choice([0, _spread(rng, 1, 32000), _spread(rng, 1, 1000000)]), 16 * rng.randint(1, 8),
                       rng.random() < 0.5, rng.random() < 0.6, rng.randrange(1 << 20))
    else:
        kind = rng.choice(["even", "mixed", "ragged"])
        hkv = rng.randint(1, 8)
        hq = hkv * rng.choice([1, 2, 3, 4, 5, 6, 8])
        batch = _spread(rng, 1, 32)
        tokens = _spread(rng, 1, 2048 // batch)
        cached = rng.choice([0, _spread(rng, 1, 30000)])
        room = (1 << 31) // (batch * hq * tokens)       # what the plain form's scores take at most
        cached = max(0, min(cached, room - tokens, (1 << 18) // batch))
        case = _attend("", rng.choice(["bf16", "f16"]), hq, hkv, kind, batch, tokens, cached, rng.randrange(1 << 20))
    del case["name"]
    return case


def _lengths(case):
    """New tokens and rows cached before them, for each sequence of a ragged batch."""
    r = random.Random(case["mix"])
    tokens, cached = case["tokens"], case["cached"]
    got = []
    for b in range(case["batch"]):
        if case["kind"] == "even":
            n, c = tokens, cached
        elif case["kind"] == "mixed":                     # one chunk, the others decode
            n, c = (tokens, cached // 2) if b == 0 else (1, r.randint(0, cached))
        else:                                             # some sequences bring nothing in this step
            n, c = (tokens if b == 0 else r.randint(0, tokens)), (cached if b == 0 else r.randint(0, cached))
        got.append((n, c))
    return got


def work(case):
    size, hq, hkv = SIZES[case["dtype"]], case["hq"], case["hkv"]
    if case["op"] == "qk_norm_rope":
        n = case["batch"] * case["length"] * (hq + hkv) * case["dim"]
        return {"bytes": 2 * n * size + 4 * case["length"], "flops": 8 * n}
    both = _lengths(case)
    tokens = sum(n for n, _ in both)
    if case["op"] == "rope_append":
        n = tokens * (hq + 2 * hkv) * HEAD
        pages = sum((n + c + PAGE - 1) // PAGE - c // PAGE for n, c in both)
        return {"bytes": 2 * n * size + 4 * (pages + 2 * len(both) + 1), "flops": 8 * tokens * (hq + hkv) * HEAD}
    seen = sum(n * c + n * (n + 1) // 2 for n, c in both)
    rows = sum(n + c for n, c in both if n)
    return {"bytes": 2 * tokens * hq * HEAD * size + 2 * rows * hkv * HEAD * size + 4 * (rows // PAGE + 3 * len(both)),
            "flops": 4 * HEAD * hq * seen}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------

def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def prepare(case, seed):
    dev, dtype = _device(), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    hq, hkv = case["hq"], case["hkv"]
    state = dict(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    def weights(dim):
        """The norm's weights and the rotation's frequencies, as a model's parameters hold them."""
        state["inv_freq"] = 10000.0 ** (-torch.arange(0, state["rot"], 2, device=dev, dtype=torch.float32) / state["rot"])
        state["wq"] = state["wk"] = None
        if state["norm"]:
            state["wq"] = (1 + 0.2 * torch.randn(dim, generator=gen, device=dev)).to(dtype)
            state["wk"] = (1 + 0.2 * torch.randn(dim, generator=gen, device=dev)).to(dtype)

    if case["op"] == "qk_norm_rope":
        b, s, d = case["batch"], case["length"], case["dim"]
        weights(d)
        x = normal(b, s, (hq + 2 * hkv) * d)              # the projection's output: queries, keys, values side by side
        state["q"] = x[..., :hq * d].view(b, s, hq, d)
        state["k"] = x[..., hq * d:(hq + hkv) * d].view(b, s, hkv, d)
        state["positions"] = torch.arange(s, device=dev, dtype=torch.int32) + int(torch.randint(0, 4096, (1,), generator=gen, device=dev))
        state["q_out"] = torch.zeros((b, hq, s, d), device=dev, dtype=dtype)
        state["k_out"] = torch.zeros((b, hkv, s, d), device=dev, dtype=dtype)
        return state

    both = _lengths(case)
    batch, tokens = len(both), sum(n for n, _ in both)
    rows = tokens + 3                                     # a padded batch: three rows behind the last sequence
    lens = [n + c for n, c in both]
    # pages of the cache are dealt in random order; an append touches few pages of a long sequence, so only the table
    # is as long as the sequence and all but the last pages are one shared page
    width = max(1, max((n + PAGE - 1) // PAGE for n in lens))
    shared = case["op"] == "rope_append"
    need = [((n + PAGE - 1) // PAGE - c0 // PAGE) if shared else (n + PAGE - 1) // PAGE for n, (_, c0) in zip(lens, both)]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)
    table = torch.full((batch, width), -1, device="cpu", dtype=torch.int32)
    order_host, at = order.cpu(), 1
    for b, (n, _) in enumerate(zip(lens, both)):
        last = (n + PAGE - 1) // PAGE
        table[b, :last] = order_host[0]
        table[b, last - need[b]:last] = order_host[at:at + need[b]]
        at += need[b]
    state["block_table"] = table.to(dev)
    state["cu_seqlens"] = torch.tensor([0] + [sum(n for n, _ in both[:b + 1]) for b in range(batch)], device=dev, dtype=torch.int32)
    state["seq_lens"] = torch.tensor(lens, device=dev, dtype=torch.int32)
    state["most"] = max(n for n, _ in both)
    state["tokens_in_all"] = tokens
    state["k_pages"] = normal(pool, hkv, PAGE, HEAD)
    state["v_pages"] = normal(pool, hkv, PAGE, HEAD)
    if case["op"] == "attn_paged":
        state["q"] = normal(rows, hq, HEAD)
        state["out"] = torch.zeros_like(state["q"])
        return state
    weights(HEAD)
    x = normal(rows, (hq + 2 * hkv) * HEAD)
    state["q"] = x[:, :hq * HEAD].view(rows, hq, HEAD)
    state["k"] = x[:, hq * HEAD:(hq + hkv) * HEAD].view(rows, hkv, HEAD)
    state["v"] = x[:, (hq + hkv) * HEAD:].view(rows, hkv, HEAD)
    state["q_out"] = torch.zeros((rows, hq, HEAD), device=dev, dtype=dtype)
    return state


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------

_kept = {}         # the framework's module and its scratch memory, which a program keeps for all its calls


def _framework():
    if "runtime" not in _kept:
        if "mlir-toy_b200" not in sys.path:
            sys.path.insert(1, "mlir-toy_b200")           # where this repository keeps its package
        from neptune_mlir import runtime

        _kept["runtime"] = runtime
    return _kept["runtime"]


def _scratch(runtime, dev):
    if dev not in _kept:
        _kept[dev] = torch.empty(runtime.attn_paged_workspace_bytes(), dtype=torch.uint8, device=dev)
    return _kept[dev]


def run(state):
    if own:
        runtime = _framework()
        if state["op"] == "qk_norm_rope":
            runtime.qk_norm_rope(state["q"], state["k"], state["positions"], state["inv_freq"], state["q_out"],
                                 state["k_out"], state["wq"], state["wk"], B=state["batch"], S=state["length"],
                                 Hq=state["hq"], Hkv=state["hkv"], D=state["dim"], rot_dim=state["rot"],
                                 interleaved=state["neighbours"], eps=EPS, dtype=state["dtype"])
            return state["q_out"], state["k_out"]
        facts = {"T": state["q"].shape[0], "B": state["batch"], "Hq": state["hq"], "Hkv": state["hkv"],
                 "max_pages": state["block_table"].shape[1], "page_size": PAGE, "D": HEAD, "dtype": state["dtype"]}
        if state["op"] == "rope_append":
            runtime.rope_append(state["q"], state["k"], state["v"], state["k_pages"], state["v_pages"],
                                state["block_table"], state["cu_seqlens"], state["seq_lens"], state["inv_freq"],
                                state["q_out"], state["wq"], state["wk"], rot_dim=state["rot"],
                                interleaved=state["neighbours"], eps=EPS, **facts)
            return state["q_out"], state["k_pages"], state["v_pages"]
        runtime.attn_paged(state["q"], state["k_pages"], state["v_pages"], state["block_table"], state["cu_seqlens"],
                           state["seq_lens"], _scratch(runtime, state["q"].device), state["out"],
                           scale_log2=math.log2(math.e) / math.sqrt(HEAD), **facts)
        return state["out"]
    return {"qk_norm_rope": _plain_rotate, "rope_append": _plain_append, "attn_paged": _plain_attend}[state["op"]](state)


def _norm_rotate(x, w, angles, rot, neighbours):
    """x [..., heads, D] with its norm and the first `rot` of D rotated by `angles` [..., rot / 2], in 32 bits."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
    c, s = angles.cos().float().unsqueeze(-2), angles.sin().float().unsqueeze(-2)
    if neighbours:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, y[..., rot:]), -1)


def _plain_rotate(state):
    angles = state["positions"].double()[:, None] * state["inv_freq"].double()
    for x, w, out in (("q", "wq", "q_out"), ("k", "wk", "k_out")):
        y = _norm_rotate(state[x], state[w], angles, state["rot"], state["neighbours"])
        state[out].copy_(y.transpose(1, 2))
    return state["q_out"], state["k_out"]


def _tokens(state):
    """For each token of the batch its sequence and its slot there."""
    cu = state["cu_seqlens"].long()
    t = torch.arange(state["tokens_in_all"], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, state["seq_lens"].long()[b] - cu[b + 1] + t


def _plain_append(state):
    b, slot = _tokens(state)
    n = state["tokens_in_all"]
    angles = slot.double()[:, None] * state["inv_freq"].double()
    dtype = state["q"].dtype
    q = _norm_rotate(state["q"][:n], state["wq"], angles, state["rot"], state["neighbours"])
    k = _norm_rotate(state["k"][:n], state["wk"], angles, state["rot"], state["neighbours"])
    state["q_out"][:n] = q.to(dtype)
    page = state["block_table"][b, slot // PAGE].long()
    state["k_pages"][page, :, slot % PAGE] = k.to(dtype)
    state["v_pages"][page, :, slot % PAGE] = state["v"][:n]
    return state["q_out"], state["k_pages"], state["v_pages"]


def _plain_attend(state):
    cu, lens = state["cu_seqlens"].long(), state["seq_lens"].long()
    new = cu[1:] - cu[:-1]
    batch, hq, hkv, most, dev = state["batch"], state["hq"], state["hkv"], state["most"], cu.device
    pages = state["block_table"].long().clamp(min=0)

    def rows(pool):                                       # [batch, hkv, rows, D], the rows behind a sequence's end cleared
        x = pool[pages].permute(0, 2, 1, 3, 4).flatten(2, 3).float()
        return x.masked_fill(torch.arange(x.shape[2], device=dev)[None, None, :, None] >= lens[:, None, None, None], 0.0)

    k, v = rows(state["k_pages"]), rows(state["v_pages"])
    i = torch.arange(most, device=dev)
    at = (cu[:-1, None] + i).clamp(max=state["q"].shape[0] - 1)
    q = state["q"][at].float().view(batch, most, hkv, hq // hkv, HEAD).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(HEAD)).view(batch, hkv, hq // hkv, most, -1)
    last = (lens - new)[:, None] + i                      # the last row that a token sees: its own
    hidden = torch.arange(x.shape[-1], device=dev) > last[:, :, None]
    x.masked_fill_(hidden[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    x.div_(x.sum(-1, keepdim=True))
    o = torch.matmul(x.flatten(2, 3), v).view(batch, hkv, hq // hkv, most, HEAD).permute(0, 3, 1, 2, 4).flatten(2, 3)
    b, slot = _tokens(state)
    state["out"][:state["tokens_in_all"]] = o[b, slot - (lens - new)[b]].to(state["out"].dtype)
    return state["out"]


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def _turn64(x, w, position, inv_freq, neighbours):
    """One norm and rotation by the definition, x [n, heads, D], position [n]: pairs as complex numbers times e^(i a)."""
    x = x.double().clone()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
    half = inv_freq.shape[0]
    first = torch.arange(half, device=x.device) * (2 if neighbours else 1)
    second = first + (1 if neighbours else half)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), position.double()[:, None] * inv_freq.double())
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None, :]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "qk_norm_rope":
        got = []
        for x, w in (("q", "wq"), ("k", "wk")):
            y = [_turn64(part, state[w], state["positions"], state["inv_freq"], case["neighbours"]) for part in state[x]]
            got.append(torch.stack(y).transpose(1, 2))
        return tuple(got)
    cu, lens, table = state["cu_seqlens"].tolist(), state["seq_lens"].tolist(), state["block_table"].tolist()
    if case["op"] == "rope_append":
        q_out, kp, vp = (state[x].double() for x in ("q_out", "k_pages", "v_pages"))
        for b, length in enumerate(lens):
            part = slice(cu[b], cu[b + 1])
            n = cu[b + 1] - cu[b]
            where = torch.arange(length - n, length, device=q_out.device)
            q_out[part] = _turn64(state["q"][part], state["wq"], where, state["inv_freq"], case["neighbours"])
            k = _turn64(state["k"][part], state["wk"], where, state["inv_freq"], case["neighbours"])
            at = 0
            while at < n:                                 # page by page
                slot = length - n + at
                take = min(n - at, PAGE - slot % PAGE)
                page, row = table[b][slot // PAGE], slot % PAGE
                kp[page, :, row:row + take] = k[at:at + take].transpose(0, 1)
                vp[page, :, row:row + take] = state["v"][cu[b] + at:cu[b] + at + take].double().transpose(0, 1)
                at += take
        return q_out, kp, vp
    if work(case)["flops"] > 4e12:
        return None
    out = state["out"].double()
    group = case["hq"] // case["hkv"]
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        use = torch.tensor(table[b][:(length + PAGE - 1) // PAGE], device=out.device)
        sees = torch.ones((n, length), dtype=torch.bool, device=out.device).tril(length - n)
        for h in range(case["hkv"]):
            k = state["k_pages"][use, h].reshape(-1, HEAD)[:length].double()
            v = state["v_pages"][use, h].reshape(-1, HEAD)[:length].double()
            for j in range(h * group, (h + 1) * group):
                x = state["q"][cu[b]:cu[b + 1], j].double() @ k.T / math.sqrt(HEAD)
                e = torch.where(sees, torch.exp(x - torch.where(sees, x, -math.inf).max(-1, keepdim=True).values), 0.0)
                out[cu[b]:cu[b + 1], j] = (e @ v) / e.sum(-1, keepdim=True)
    return out
