"""Cases of the serving-step operators: writing a paged K/V cache, reading it
back, attention of new tokens over it, and rules on logits with the greedy
choice. Each case runs in a plain form (elementary torch operations in 32 bits)
or through this package's operators (`own`)."""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


# ---------------------------------------------------------------------------
# Cases

def _attend(name, seqs, new, ctx, q_heads, kv_heads, dim, page, type, format, causal=True, mix=0):
    return {"name": name, "op": "attend", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page, "type": type,
            "format": format, "causal": causal, "mix": mix}


def _move(name, op, seqs, new, ctx, kv_heads, dim, page, type, format, mix=0):
    return {"name": name, "op": op, "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "kv_heads": kv_heads, "dim": dim, "page": page, "type": type, "format": format,
            "mix": mix}


def _logits(name, rows, vocab, type, history, bias, grammar, adjusted, mix=0):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "type": type, "history": history,
            "bias": bias, "grammar": grammar, "adjusted": adjusted, "mix": mix}


def listed():
    return [
        # One decode step of 64 sequences: a token each, the activations in f32 as the decoder has them,
        # into an f16 cache (16 heads of 64, the 600M decoder).
        _move("write_step", "write", 64, (1, 1), (20, 200), 16, 64, 16, "f32", "f16", 1),
        # Prompts of a batch into an 8-bit cache and back (16 heads of 128, the 3.3B decoder).
        _move("write_prompts", "write", 24, (150, 1900), (200, 2000), 16, 128, 64, "bf16", "q8", 2),
        # One short sequence read back, as when it moves to another worker.
        _move("read_one", "read", 1, (77, 77), (77, 77), 16, 64, 16, "f16", "f16", 3),
        # A batch's long 8-bit sequences read back for another cache.
        _move("read_batch", "read", 16, (900, 9000), (900, 9000), 8, 128, 64, "f16", "q8", 4),
        # The latency of one sentence: one token over 33 positions, f32 activations over the f16 cache.
        _attend("step_one", 1, (1, 1), (33, 33), 16, 16, 64, 16, "f32", "f16", True, 5),
        # The ordinary decode step of a server: 64 sentences of all lengths.
        _attend("step_batch", 64, (1, 1), (24, 1024), 16, 16, 64, 32, "f16", "q8", True, 6),
        # Decode over long documents with shared heads.
        _attend("step_long", 8, (1, 1), (20000, 65000), 32, 8, 128, 64, "bf16", "q8", True, 7),
        # A few tokens a sequence: drafts being checked, forced prefixes.
        _attend("few_tokens", 16, (2, 7), (100, 3000), 16, 4, 128, 16, "f16", "f16", True, 8),
        # Continuous batching: decoding sequences and prompt chunks in one call.
        _attend("mixed_chunks", 12, (1, 700), (700, 9000), 16, 16, 128, 64, "bf16", "f16", True, 9),
        # The largest: a chunk of a long document's prompt.
        _attend("long_chunk", 1, (4099, 4099), (20011, 20011), 16, 16, 128, 64, "f16", "q8", True, 10),
        # One sentence's step: the choice among 256206 tokens under a repetition penalty.
        _logits("choose_one", 1, 256206, "f32", 60, 0, 0, False, 11),
        # A batch's step with every rule, adjusted logits kept for sampling or a beam.
        _logits("rules_batch", 64, 256206, "f32", 200, 40, 5, True, 12),
    ]


_MOST = {"write": (1.1e9, 1e15), "read": (4e8, 1e15), "attend": (5e8, 5.5e11), "logits": (1.2e8, 1e15)}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges; drawn anew while it would cost more than the largest of its operator."""
    while True:
        op = rng.choice(["attend", "attend", "attend", "write", "read", "logits"])
        mix = rng.randrange(1 << 20)
        if op == "logits":
            case = _logits("", _log_int(rng, 1, 96), _log_int(rng, 4000, 256206), rng.choice(["f32", "f16", "bf16"]),
                           _log_int(rng, 1, 1000), rng.choice([0, _log_int(rng, 1, 100)]),
                           rng.choice([0, rng.randint(1, 8)]), rng.random() < 0.5, mix)
        else:
            dim, page = rng.choice([64, 64, 128, 128, 32, 16]), rng.choice([16, 32, 64, 128])
            format = rng.choice(["f16", "q8"])
            if op == "attend":
                kv_heads = rng.choice([16, 8, 4, 2, 1])
                q_heads = kv_heads * rng.choice([1, 1, 2, 4, 7, 8])
                kind = rng.choice(["step", "step", "few", "chunk", "chunk"])
                causal = rng.random() < 0.8
                seqs = _log_int(rng, 1, 96 if kind != "chunk" else 16)
                new = {"step": (1, 1), "few": (2, 8), "chunk": (rng.choice([1, 16, 100]), _log_int(rng, 100, 4100))}[kind]
                lo = max(new[1], _log_int(rng, 8, 8000))
                ctx = (lo, lo + _log_int(rng, 1, 30000))
                # f32 activations are the decoder's own; long chunks come from 16-bit ones
                type = rng.choice(["f32", "f16", "bf16"] if kind != "chunk" else ["f16", "bf16"])
                case = _attend("", seqs, new, ctx, q_heads, kv_heads, dim, page, type, format, causal, mix)
            else:
                kv_heads = rng.choice([16, 16, 8, 4, 12])
                seqs = _log_int(rng, 1, 96)
                hi = 1 if op == "write" and rng.random() < 0.4 else _log_int(rng, 2, 9000)
                new = (max(1, hi // rng.choice([1, 2, 9])), hi)
                ctx = (new[1], new[1] + _log_int(rng, 1, 400))
                case = _move("", op, seqs, new, ctx, kv_heads, dim, page, rng.choice(["f32", "f16", "bf16"]), format,
                             mix)
        del case["name"]
        w = work(case)
        most = _MOST[op]
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and _pool_bytes(case) < 3e9:
            return case


def _lengths(case):
    """New tokens and positions (new ones included) of every sequence, from the case alone."""
    rng = random.Random(case["mix"])
    new = [_log_int(rng, case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    ctx = [max(n, _log_int(rng, case["ctx_lo"], case["ctx_hi"])) for n in new]
    return new, ctx


def _pool_pages(case):
    _, ctx = _lengths(case)
    return sum(-(-c // case["page"]) for c in ctx) + 3


def _row_bytes(case):
    """Bytes of one position of one head of K or V in the cache."""
    return case["dim"] * 2 if case["format"] == "f16" else case["dim"] + 4


def _pool_bytes(case):
    if case["op"] == "logits":
        return 0
    return 2 * _pool_pages(case) * case["page"] * case["kv_heads"] * _row_bytes(case)


def work(case):
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        b = n * SIZE[case["type"]] * (2 if case["adjusted"] else 1) + case["rows"] * (case["history"] * 4 + 12)
        b += case["rows"] * case["bias"] * 8 + case["grammar"] * ((case["vocab"] + 31) // 32) * 4
        return {"bytes": float(b), "flops": 4.0 * n}
    new, ctx = _lengths(case)
    table = 4 * sum(-(-c // case["page"]) for c in ctx) + 8 * len(new)
    if case["op"] == "attend":
        pairs = sum(n * c - (n * (n - 1) // 2 if case["causal"] else 0) for n, c in zip(new, ctx))
        kv = 2 * sum(ctx) * case["kv_heads"] * _row_bytes(case)
        io = 2 * sum(new) * case["q_heads"] * case["dim"] * SIZE[case["type"]]
        return {"bytes": float(kv + io + table), "flops": 4.0 * pairs * case["q_heads"] * case["dim"]}
    rows = sum(new) * case["kv_heads"]
    b = 2 * rows * (case["dim"] * SIZE[case["type"]] + _row_bytes(case)) + table
    if case["op"] == "write" and case["format"] == "q8":
        b += 2 * rows * case["dim"] * 4  # the values that the codes stand for, read back
    return {"bytes": float(b), "flops": 4.0 * rows * case["dim"]}


# ---------------------------------------------------------------------------
# Inputs

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _kv_like(gen, *shape):
    """Rows as projections give them: normal, rows of unlike size, some channels larger."""
    x = _normal(gen, *shape)
    x *= torch.exp(0.3 * _normal(gen, *shape[:-1], 1))
    x[..., :: 16] *= 3.0
    return x


def _q8(x):
    """Codes and scales of rows x (f32): d = max|x| / 127, code = x / d to the nearest whole number."""
    d = x.abs().amax(-1) / torch.full((), 127.0, device=x.device).expand(x.shape[:-1])
    code = torch.where(d[..., None] > 0, torch.round(x / d[..., None]), torch.zeros_like(x))
    return code.to(torch.int8), d


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 7919 + 13)
    state = {"case": case}
    if case["op"] == "logits":
        return _prepare_logits(case, seed, gen, state)
    H, D, page = case["kv_heads"], case["dim"], case["page"]
    new, ctx = _lengths(case)
    pages = _pool_pages(case)
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.zeros((len(new), max(-(-c // page) for c in ctx)), np.int32)
    at = 0
    for b, c in enumerate(ctx):
        n = -(-c // page)
        table[b, :n] = order[at: at + n]
        at += n
    k, v, ks, vs = [], [], [], []
    step = max(1, (64 << 20) // (H * page * D))
    for p0 in range(0, pages, step):  # the cache holds what earlier steps wrote, unused slots included
        n = min(step, pages - p0)
        for data, scale in ((k, ks), (v, vs)):
            x = _kv_like(gen, n, H, page, D)
            if case["format"] == "q8":
                code, d = _q8(x)
                data.append(code)
                scale.append(d)
            else:
                data.append(x.half())
    state["k"], state["v"] = torch.cat(k), torch.cat(v)
    state["k_scale"] = torch.cat(ks) if ks else None
    state["v_scale"] = torch.cat(vs) if vs else None
    state["new"], state["ctx"] = new, ctx
    state["table"] = torch.from_numpy(table).to(DEV)
    state["q_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(DEV)
    state["kv_len"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    tokens, dtype = sum(new), TYPES[case["type"]]
    if case["op"] == "attend":
        state["q"] = (2.0 * _normal(gen, tokens, case["q_heads"], D)).to(dtype)
    if case["op"] == "write":  # K and V as slices of one projection's rows
        both = _kv_like(gen, tokens, 2, H, D).to(dtype)
        state["k_new"], state["v_new"] = both[:, 0], both[:, 1]
    if own:
        from malaga_b200 import ops

        state["cache"] = ops.PagedKV(state["k"], state["v"], state["k_scale"], state["v_scale"])
        state["seqs"] = ops.Seqs(state["table"], state["q_start"], state["kv_len"], max_new=max(new), max_len=max(ctx),
                                 tokens=tokens)
    return state


def _prepare_logits(case, seed, gen, state):
    rows, vocab = case["rows"], case["vocab"]
    rng = np.random.default_rng(seed)
    logits = 2.0 * _normal(gen, rows, vocab)
    # tokens already said are likely ones, some said more than once
    hist = np.minimum(rng.zipf(1.2, (rows, case["history"])), vocab) - 1
    hist = (hist * 7919 + 13) % vocab
    hist_len = rng.integers((case["history"] + 1) // 2, case["history"] + 1, rows)
    said = torch.from_numpy(hist).to(DEV)
    logits.scatter_add_(1, said, 3.0 * torch.rand(said.shape, generator=gen, device=DEV))
    state["logits"] = logits.to(TYPES[case["type"]])
    state["history"] = torch.from_numpy(hist.astype(np.int32)).to(DEV)
    state["history_len"] = torch.from_numpy(hist_len.astype(np.int32)).to(DEV)
    state["repetition"] = torch.from_numpy(rng.uniform(1.0, 1.5, rows).astype(np.float32)).to(DEV)
    state["frequency"] = torch.from_numpy(rng.uniform(0.0, 0.5, rows).astype(np.float32)).to(DEV)
    state["presence"] = torch.from_numpy(rng.uniform(0.0, 0.5, rows).astype(np.float32)).to(DEV)
    state["bias_ids"] = state["bias"] = state["allow"] = state["allow_row"] = None
    if case["bias"]:
        ids = np.stack([rng.choice(vocab, case["bias"], replace=False) for _ in range(rows)])
        state["bias_ids"] = torch.from_numpy(ids.astype(np.int32)).to(DEV)
        state["bias"] = torch.from_numpy(rng.normal(0.0, 3.0, ids.shape).astype(np.float32)).to(DEV)
    if case["grammar"]:
        share = torch.rand(case["grammar"], 1, generator=gen, device=DEV) ** 3 * 0.9 + 0.01
        words = (vocab + 31) // 32
        bits = torch.rand(case["grammar"], words * 32, generator=gen, device=DEV) < share
        weight = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], device=DEV)
        state["allow"] = (bits.view(-1, words, 32) * weight).sum(-1).to(torch.int32)
        # a row follows one of the grammars or, as -1, none
        state["allow_row"] = torch.from_numpy(rng.integers(-1, case["grammar"], rows).astype(np.int32)).to(DEV)
    if own:
        from malaga_b200 import ops

        state["rules"] = ops.LogitRules(
            history=state["history"], history_len=state["history_len"], repetition=state["repetition"],
            frequency=state["frequency"], presence=state["presence"], bias_ids=state["bias_ids"], bias=state["bias"],
            allow=state["allow"], allow_row=state["allow_row"])
    return state


# ---------------------------------------------------------------------------
# One pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case = state["case"]
    if case["op"] == "write":
        state["cache"].write(state["seqs"], state["k_new"], state["v_new"])
        if case["format"] == "q8":
            return state["cache"].read(state["seqs"], torch.float32)
        return state["k"], state["v"]
    if case["op"] == "read":
        return state["cache"].read(state["seqs"], TYPES[case["type"]])
    if case["op"] == "attend":
        return state["cache"].attend(state["seqs"], state["q"], causal=case["causal"])
    if case["adjusted"]:
        return state["rules"].choose(state["logits"], adjusted=torch.empty_like(state["logits"]))
    return state["rules"].choose(state["logits"])


def _slots(state, b):
    """Page and place in it of every position of sequence b."""
    page = state["k"].shape[2]
    pos = torch.arange(state["ctx"][b], device=DEV)
    return state["table"][b][pos // page].long(), pos % page


def _rows_plain(state, which, at, place):
    """Rows [n, heads, dim] of the cache in f32."""
    x = state[which][at, :, place].float()
    if state[which + "_scale"] is not None:
        x = x * state[which + "_scale"][at, :, place][..., None]
    return x


def _run_plain(state):
    case = state["case"]
    if case["op"] == "write":
        return _write_plain(state)
    if case["op"] == "read":
        out = []
        for which in "kv":
            parts = []
            for b, n in enumerate(state["new"]):
                at, place = _slots(state, b)
                parts.append(_rows_plain(state, which, at[-n:], place[-n:]))
            out.append(torch.cat(parts).to(TYPES[case["type"]]))
        return tuple(out)
    if case["op"] == "attend":
        return _attend_plain(state)
    return _logits_plain(state)


def _write_plain(state):
    slots = [_slots(state, b) for b in range(len(state["new"]))]
    at = torch.cat([a[-n:] for (a, _), n in zip(slots, state["new"])])
    place = torch.cat([p[-n:] for (_, p), n in zip(slots, state["new"])])
    out = []
    for which in "kv":
        x = state[which + "_new"].float()
        if state["case"]["format"] == "q8":
            code, d = _q8(x)
            state[which][at, :, place] = code
            state[which + "_scale"][at, :, place] = d
            out.append(_rows_plain(state, which, at, place))
        else:
            state[which][at, :, place] = x.half()
            out.append(state[which])
    return tuple(out)


def _attend_plain(state):
    case = state["case"]
    H, D, group = case["kv_heads"], case["dim"], case["q_heads"] // case["kv_heads"]
    out, t0 = torch.empty_like(state["q"]), 0
    for b, n in enumerate(state["new"]):
        length = state["ctx"][b]
        at, place = _slots(state, b)
        k, v = _rows_plain(state, "k", at, place), _rows_plain(state, "v", at, place)
        q = state["q"][t0: t0 + n].float().view(n, H, group, D)
        for h in range(0, H, max(1, int(2e8 // (n * group * length)))):
            hs = slice(h, h + max(1, int(2e8 // (n * group * length))))
            s = torch.einsum("nhgd,lhd->hgnl", q[:, hs], k[:, hs]) * (D ** -0.5)
            if case["causal"]:
                pos = torch.arange(length - n, length, device=DEV)
                s = s.masked_fill(torch.arange(length, device=DEV)[None] > pos[:, None], -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.einsum("hgnl,lhd->hgnd", p, v[:, hs]) / p.sum(-1, keepdim=True)
            out[t0: t0 + n].view(n, H, group, D)[:, hs] = o.permute(2, 0, 1, 3).to(out.dtype)
        t0 += n
    return out


def _logits_plain(state):
    case = state["case"]
    y = state["logits"].float()
    live = torch.arange(state["history"].shape[1], device=DEV)[None] < state["history_len"][:, None]
    count = torch.zeros_like(y).scatter_add_(1, state["history"].long(), live.float())
    r = state["repetition"][:, None]
    y = torch.where(count > 0, torch.where(y > 0, y / r, y * r), y)
    y = y - torch.where(count > 0, state["frequency"][:, None] * count + state["presence"][:, None], 0.0)
    if state["bias"] is not None:
        y = y.scatter_add(1, state["bias_ids"].long(), state["bias"])
    if state["allow"] is not None:
        bit = torch.arange(32, device=DEV, dtype=torch.int32)
        allow = ((state["allow"][:, :, None] >> bit) & 1).bool().flatten(1)[:, : y.shape[1]]
        y = y.masked_fill((state["allow_row"][:, None] >= 0) & ~allow[state["allow_row"].clamp(min=0).long()], -math.inf)
    top = y.amax(1, keepdim=True)
    where = torch.arange(y.shape[1], device=DEV, dtype=torch.int32)[None]
    ids = torch.where(y == top, where, y.shape[1]).amin(1).to(torch.int32)
    logp = -torch.log(torch.exp(y - top).sum(1))
    return (ids, logp, y.to(state["logits"].dtype)) if case["adjusted"] else (ids, logp)


# ---------------------------------------------------------------------------
# The definitions in 64 bits

def _stored(state, which, x):
    """64-bit values that rows x stand for once stored; the scale of 8-bit codes is held in 32 bits and the quotient
    is the 32-bit one, which is part of the format."""
    if state["case"]["format"] == "f16":
        return x
    d = (x.abs().amax(-1, keepdim=True) / 127.0).float().double()
    ratio = (x / torch.where(d > 0, d, 1.0)).float().double()
    return torch.where(d > 0, torch.round(ratio), 0.0) * d


def _position_rows(state, which, b):
    """Positions of sequence b in 64 bits, [heads, positions, dim]."""
    pages = state["table"][b, : -(-state["ctx"][b] // state["case"]["page"])].long()
    x = state[which].index_select(0, pages).double()
    if state["case"]["format"] == "q8":
        x *= state[which + "_scale"].index_select(0, pages).double().unsqueeze(-1)
    return x.transpose(0, 1).flatten(1, 2)[:, : state["ctx"][b]]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(case, state)
    if case["op"] == "read":
        return tuple(torch.cat([_position_rows(state, w, b)[:, -n:].transpose(0, 1)
                                for b, n in enumerate(state["new"])]) for w in "kv")
    if case["op"] == "write":
        out = []
        for which in "kv":
            rows = _stored(state, which, state[which + "_new"].double())
            if case["format"] == "f16":
                # the cache seen as one row of heads for every place, a sequence's new rows put in by their place's number
                pool = state[which].double().transpose(1, 2).flatten(0, 1).clone()
                for b, part in enumerate(rows.split(state["new"])):
                    place = np.arange(state["ctx"][b] - len(part), state["ctx"][b])
                    number = state["table"][b].cpu().numpy()[place // case["page"]].astype(np.int64) * case["page"]
                    pool[torch.from_numpy(number + place % case["page"]).to(DEV)] = part
                rows = pool.unflatten(0, (-1, case["page"])).transpose(1, 2)
            out.append(rows)
        return tuple(out)
    n_all, group = sum(state["new"]), case["q_heads"] // case["kv_heads"]
    out, t = torch.zeros(n_all, case["q_heads"], case["dim"], dtype=torch.float64, device=DEV), 0
    for b, n in enumerate(state["new"]):
        keys, values = _position_rows(state, "k", b), _position_rows(state, "v", b)
        length = state["ctx"][b]
        first = length - n
        for h in range(case["q_heads"]):
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                s = state["q"][t + i: t + i + m, h].double() @ keys[h // group].T / math.sqrt(case["dim"])
                if case["causal"]:
                    s += torch.full_like(s, -math.inf).triu_(first + i + 1)
                out[t + i: t + i + m, h] = torch.softmax(s, -1) @ values[h // group]
        t += n
    return out


def _exact_logits(case, state):
    rows = []
    for r in range(case["rows"]):
        y = state["logits"][r].double()
        said, count = state["history"][r, : int(state["history_len"][r])].long().unique(return_counts=True)
        rep, freq, pres = (float(state[k][r]) for k in ("repetition", "frequency", "presence"))
        z = y[said]
        y[said] = torch.maximum(z, z * 0) / rep + torch.minimum(z, z * 0) * rep - freq * count - pres
        if case["bias"]:
            y.index_add_(0, state["bias_ids"][r].long(), state["bias"][r].double())
        if case["grammar"] and int(state["allow_row"][r]) >= 0:
            words = state["allow"][int(state["allow_row"][r])].cpu().numpy().view(np.uint8)
            bits = np.unpackbits(words, bitorder="little")[: case["vocab"]]
            y[torch.from_numpy(bits == 0).to(DEV)] = -math.inf
        rows.append(y)
    y = torch.stack(rows)
    top = y.max(1).values
    ids = torch.stack([(row == t).nonzero()[0, 0] for row, t in zip(y, top)]).to(torch.int32)
    logp = top - torch.logsumexp(y, 1)
    return (ids, logp, y) if case["adjusted"] else (ids, logp)
