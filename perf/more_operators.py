"""The operators of a step that serves several requests with drafted tokens on a paged cache, and the cases they are
measured on.

- append: a step's keys (normed, rotated) and values into the requests' pages, and its queries normed and rotated
- attend: attention of every row of the step over its request's cached tokens and its ancestors among the drafted ones
- accept: the drafted tokens that the model's own picks confirm, and their keys and values moved to consecutive slots

Row i of a request that has n tokens in the cache lies in slot n + i and at position n + depth(i); without a tree the rows
are a chain. ``run`` computes them in elementary torch operations, or with the framework's kernels where ``own`` is true.
"""
import math

import numpy as np
import torch

own = False

D = 128          # head dimension
VOCAB = 151936   # token ids (Qwen3-0.6B's vocabulary)
DEV = "cuda"


def listed():
    return [
        # a decode step of one request (Llama-3.1-8B heads): latency
        {"name": "append 1", "op": "append", "hq": 32, "hkv": 8, "page": 16, "seqs": 1, "n_lo": 2611, "n_hi": 2611,
         "t_lo": 1, "t_hi": 1, "tree": False, "norm": False, "pad": 0},
        # drafted trees of many requests, per-head norms (Qwen3-0.6B heads), a step padded for a captured graph
        {"name": "append 24 trees", "op": "append", "hq": 16, "hkv": 8, "page": 32, "seqs": 24, "n_lo": 50, "n_hi": 3500,
         "t_lo": 9, "t_hi": 45, "tree": True, "norm": True, "pad": 7},
        # pieces of three long prompts (Llama-3.1-70B heads)
        {"name": "append 3 prompts", "op": "append", "hq": 64, "hkv": 8, "page": 64, "seqs": 3, "n_lo": 0, "n_hi": 4000,
         "t_lo": 1000, "t_hi": 2500, "tree": False, "norm": False, "pad": 0},
        # a decode step early in a chat: latency
        {"name": "attend 1x611", "op": "attend", "hq": 32, "hkv": 8, "page": 16, "seqs": 1, "n_lo": 610, "n_hi": 610,
         "t_lo": 1, "t_hi": 1, "tree": False, "pad": 0},
        # a decode step of many requests of very different lengths (Qwen2.5-7B heads), padded for a captured graph
        {"name": "attend 48 ragged", "op": "attend", "hq": 28, "hkv": 4, "page": 16, "seqs": 48, "n_lo": 20, "n_hi": 9000,
         "t_lo": 1, "t_hi": 1, "tree": False, "pad": 16},
        # a decode step at the end of the longest context (Llama-3.1-8B heads)
        {"name": "attend 1x131071", "op": "attend", "hq": 32, "hkv": 8, "page": 64, "seqs": 1, "n_lo": 131070,
         "n_hi": 131070, "t_lo": 1, "t_hi": 1, "tree": False, "pad": 0},
        # one request's drafted tree behind a long prompt (Qwen2.5-7B's benchmark prompt, Llama-3.1-8B heads)
        {"name": "attend tree 64x8200", "op": "attend", "hq": 32, "hkv": 8, "page": 32, "seqs": 1, "n_lo": 8200,
         "n_hi": 8200, "t_lo": 64, "t_hi": 64, "tree": True, "pad": 0},
        # drafted trees of many requests (Llama-3.1-8B heads)
        {"name": "attend 32 trees", "op": "attend", "hq": 32, "hkv": 8, "page": 64, "seqs": 32, "n_lo": 300, "n_hi": 5000,
         "t_lo": 9, "t_hi": 45, "tree": True, "pad": 5},
        # a piece of a prompt behind its first pieces
        {"name": "attend 2049 behind 6145", "op": "attend", "hq": 32, "hkv": 8, "page": 128, "seqs": 1, "n_lo": 6145,
         "n_hi": 6145, "t_lo": 2049, "t_hi": 2049, "tree": False, "pad": 0},
        # one request's small tree (Qwen2.5-7B: 28 layers): latency
        {"name": "accept 1x8", "op": "accept", "hkv": 4, "page": 16, "layers": 28, "seqs": 1, "n_lo": 611, "n_hi": 611,
         "t_lo": 8, "t_hi": 8, "tree": True, "pad": 0},
        # trees of many requests (Qwen3-0.6B: 28 layers)
        {"name": "accept 24 trees", "op": "accept", "hkv": 8, "page": 32, "layers": 28, "seqs": 24, "n_lo": 10,
         "n_hi": 300, "t_lo": 9, "t_hi": 45, "tree": True, "pad": 7},
        # the largest trees of many requests (Llama-3.1-8B: 32 layers); long contexts change nothing for this operator
        {"name": "accept 60 trees", "op": "accept", "hkv": 8, "page": 16, "layers": 32, "seqs": 60, "n_lo": 10,
         "n_hi": 150, "t_lo": 50, "t_hi": 64, "tree": True, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "accept"])
    hq, hkv = rng.choice([(16, 8), (28, 4), (32, 8), (64, 8), (10, 10), (8, 1), (14, 2), (40, 8)])
    c = {"op": op, "hq": hq, "hkv": hkv, "page": rng.choice([16, 32, 64, 128]), "pad": rng.choice([0, rng.randint(1, 20)])}
    if op == "accept":
        del c["hq"]
        c.update(layers=rng.randint(8, 32), seqs=_log(rng, 1, 48), n_lo=_log(rng, 1, 100), tree=rng.random() < 0.8)
        c["t_lo"] = _log(rng, 2, 48)
        c.update(n_hi=c["n_lo"] + _log(rng, 1, 100), t_hi=c["t_lo"] + rng.randint(0, 16))
        return c
    if op == "append":
        c["norm"] = rng.random() < 0.4
    kind = rng.choice(["decode", "tree", "prompt"])
    c["tree"] = kind == "tree"
    if kind == "prompt":
        c.update(seqs=rng.randint(1, 3), t_lo=_log(rng, 100, 1000))
        c["t_hi"] = c["t_lo"] + _log(rng, 1, 300)
    else:
        c.update(seqs=_log(rng, 1, 64), t_lo=1 if kind == "decode" else _log(rng, 2, 40))
        c["t_hi"] = c["t_lo"] if kind == "decode" else c["t_lo"] + rng.randint(0, 24)
    # contexts up to the longest listed, bounded by the largest listed pass
    most = int(min(130000, 500e6 / (4 * D * hkv * c["seqs"]), 220e9 / (4 * D * hq * c["seqs"] * c["t_hi"]) - c["t_hi"]))
    c["n_hi"] = _log(rng, 100, max(101, most))
    c["n_lo"] = rng.choice([0, _log(rng, 1, c["n_hi"])])
    return c


# ---------------------------------------------------------------- inputs


def _lengths(case):
    """Cached tokens of each request: spread evenly over the logarithm, in no order."""
    lo, hi = math.log(case["n_lo"] + 1), math.log(case["n_hi"] + 1)
    return [int(round(math.exp(lo + ((0.5 + 0.6180339887 * s) % 1) * (hi - lo)))) - 1 for s in range(case["seqs"])]


def _rows(case):
    """Rows of each request in the step."""
    return [case["t_lo"] + int(((0.25 + 0.7548776662 * s) % 1) * (case["t_hi"] - case["t_lo"] + 1))
            for s in range(case["seqs"])]


def _accepted(case):
    """How many rows of each request will be confirmed: the first, and up to five drafted ones."""
    return [1 + int(((0.75 + 0.5698402910 * s) % 1) * min(t, 6)) if t > 1 else 1 for s, t in enumerate(_rows(case))]


def _parents(case, r):
    """Parents of every row within its request (-1: the first row) and the rows that will be confirmed. A path of drafted
    tokens runs through a random subset of the rows; the others hang from earlier rows, recent ones more often."""
    parents, paths = [], []
    for t, a in zip(_rows(case), _accepted(case)):
        if case["tree"]:
            p = (np.arange(t) * np.sqrt(r.random(t))).astype(np.int64)
            path = np.concatenate([[0], np.sort(r.permutation(np.arange(1, t))[:a - 1])])
            p[path[1:]] = path[:-1]
            p[0] = -1
        else:
            p, path = np.arange(t) - 1, np.arange(a)
        parents.append(p)
        paths.append(path)
    return parents, paths


def _rope(max_pos):
    """cos and sin of position times frequency, [max_pos, 64] FP16, as the framework's tables (theta 500000)."""
    f = 500000.0 ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64)
    a = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.cos(a).half(), torch.sin(a).half()


def _int(x):
    return torch.as_tensor(np.ascontiguousarray(x), device=DEV, dtype=torch.int32)


def prepare(case, seed):
    g, r = torch.Generator(device=DEV).manual_seed(seed), np.random.RandomState(seed % (1 << 32))
    op, hkv, page = case["op"], case["hkv"], case["page"]
    n, t = np.array(_lengths(case)), np.array(_rows(case))
    starts = np.concatenate([[0], np.cumsum(t)])
    rows = int(starts[-1]) + case["pad"]
    s = {"case": case, "rows": rows, "max_rows": int(t.max())}
    # pages in random order, a few that belong to nobody, and entries behind a request's last page that mean nothing
    need = -(-(n + t) // page)
    pages = int(need.sum()) + 3
    order, table = r.permutation(pages), np.full((len(n), int(need.max()) + 2), -1)
    for i, (m, at) in enumerate(zip(need, np.cumsum(need) - need)):
        table[i, :m] = order[at:at + m]
    s["table"], s["length"], s["row_start"] = _int(table), _int(n), _int(starts)
    parents, paths = _parents(case, r)
    s["parent"] = _int(np.concatenate(parents + [np.full(case["pad"], -1)])) if case["tree"] else None

    def pool(*layers):
        return torch.randn(*layers, pages, hkv, page, D, generator=g, device=DEV, dtype=torch.float16)

    if op == "accept":
        s["k"], s["v"] = pool(case["layers"]), pool(case["layers"])
        tokens, picks = r.randint(0, VOCAB, rows), r.randint(0, VOCAB, rows)
        for at, path in zip(starts, paths):
            picks[at + path[:-1]] = tokens[at + path[1:]]
        s["tokens"], s["picks"] = (torch.as_tensor(x, device=DEV, dtype=torch.int64) for x in (tokens, picks))
        s["out"] = {"accepted": torch.empty(len(n), s["max_rows"], device=DEV, dtype=torch.int32),
                    "n_accepted": torch.empty(len(n), device=DEV, dtype=torch.int32),
                    "next_token": torch.empty(len(n), device=DEV, dtype=torch.int64),
                    "new_length": torch.empty(len(n), device=DEV, dtype=torch.int32)}
        return s
    s["k"], s["v"] = pool(), pool()
    hq = case["hq"]
    gain = torch.exp(0.5 * torch.randn(D, generator=g, device=DEV))  # a few strong channels
    if op == "append":
        s["cos"], s["sin"] = _rope(int((n + t).max()) + 5)
        # the rows of the fused projection, as the model path has them
        qkv = torch.randn(rows, hq + 2 * hkv, D, generator=g, device=DEV) * gain
        s["qkv"] = qkv.half()
        s["norms"] = [(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).half() for _ in "qk"] if case["norm"] else None
        s["q_out"] = torch.zeros(rows, hq, D, device=DEV, dtype=torch.float16)
    else:
        s["k"] *= gain.half()
        s["q"] = torch.randn(rows, hq, D, generator=g, device=DEV).half()
        s["out"] = torch.zeros(rows, hq, D, device=DEV, dtype=torch.float16)
    return s


# ---------------------------------------------------------------- plain forms


def _where(s):
    """For the rows that belong to a request: the request, and the row's number in it."""
    starts = s["row_start"].long()
    r = torch.arange(s["rows"], device=DEV)
    r = r[:int(sum(_rows(s["case"])))]
    seq = torch.searchsorted(starts, r, right=True) - 1
    return r, seq, r - starts[seq]


def _padded(s):
    """Parents as [requests, most rows], -1 for first rows and behind a request's last."""
    r, seq, i = _where(s)
    p = torch.full((s["case"]["seqs"], s["max_rows"]), -1, device=DEV)
    p[seq, i] = i - 1 if s["parent"] is None else s["parent"][r].long()
    return p


def _lineage(s):
    """[requests, row, row]: whether the second is the first or an ancestor of it."""
    p = _padded(s)
    m = p.shape[1]
    if s["parent"] is None:
        return torch.ones(m, m, dtype=torch.bool, device=DEV).tril().expand(p.shape[0], m, m)
    a = torch.eye(m, device=DEV).expand(p.shape[0], m, m) + (p[:, :, None] == torch.arange(m, device=DEV)).float()
    for _ in range(max(1, (m - 1).bit_length())):  # ancestors up to twice as far each time
        a = (a @ a).clamp(max=1)
    return a > 0


def _slots(s, seq, j):
    """Page and place in it of slots j of requests seq."""
    page = s["case"]["page"]
    return s["table"][seq, torch.div(j, page, rounding_mode="floor")].long(), j % page


def _plain_append(s):
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    r, seq, i = _where(s)
    depth = _lineage(s).sum(2)[seq, i] - 1 if s["parent"] is not None else i
    slot, pos = s["length"].long()[seq] + i, s["length"].long()[seq] + depth
    x = s["qkv"][r].float()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], s["qkv"][r, hq + hkv:]
    if s["norms"] is not None:
        q, k = (y * torch.rsqrt((y * y).mean(2, keepdim=True) + 1e-6) * w.float() for y, w in zip((q, k), s["norms"]))
    c, sn = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]
    q, k = (torch.cat([y[..., :64] * c - y[..., 64:] * sn, y[..., 64:] * c + y[..., :64] * sn], 2) for y in (q, k))
    page, place = _slots(s, seq, slot)
    s["k"][page, :, place] = k.half()
    s["v"][page, :, place] = v
    s["q_out"][r] = q.half()
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_attend(s):
    case = s["case"]
    hq, hkv, seqs = case["hq"], case["hkv"], case["seqs"]
    r, seq, i = _where(s)
    n = s["length"].long()
    m = s["max_rows"]
    most = max(a + b for a, b in zip(_lengths(case), _rows(case)))
    j = torch.arange(most, device=DEV)
    page, place = _slots(s, torch.arange(seqs, device=DEV)[:, None], j[None])
    k, v = (s[x][page.clamp(min=0), :, place].permute(0, 2, 1, 3).float() for x in ("k", "v"))  # [request, head, slot, D]
    q = torch.zeros(seqs, m, hq, D, device=DEV)
    q[seq, i] = s["q"][r].float()
    q = q.reshape(seqs, m, hkv, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, D)
    x = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(D)).reshape(seqs, hkv, m, -1, most)
    node = j - n[:, None]  # [request, slot]: the row whose key lies there, or below 0: cached before
    see = torch.gather(_lineage(s), 2, node.clamp(0, m - 1)[:, None].expand(seqs, m, most)) | (node < 0)[:, None]
    see = see & (node < (s["row_start"][1:] - s["row_start"][:-1]).long()[:, None])[:, None]
    x.masked_fill_(~see[:, None, :, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_().masked_fill_(~see[:, None, :, None], 0)
    z = x.sum(-1, keepdim=True)
    v = v.masked_fill((node >= (s["row_start"][1:] - s["row_start"][:-1]).long()[:, None])[:, None, :, None], 0)
    o = (x.reshape(seqs, hkv, -1, most) @ v).reshape(seqs, hkv, m, -1, D) / z
    s["out"][r] = o.permute(0, 2, 1, 3, 4).reshape(seqs, m, hq, D)[seq, i].half()
    return {"out": s["out"]}


def _plain_accept(s):
    case, o = s["case"], s["out"]
    r, seq, i = _where(s)
    m = s["max_rows"]
    p = _padded(s)
    token = torch.full_like(p, -1)
    pick = torch.full_like(p, -2)
    token[seq, i], pick[seq, i] = s["tokens"][r], s["picks"][r]
    # a row holds when it is the lowest of its parent's children with the parent's pick, and so are all its ancestors
    fits = (p >= 0) & (token == torch.gather(pick, 1, p.clamp(min=0)))
    twins = fits[:, :, None] & fits[:, None, :] & (p[:, :, None] == p[:, None, :])
    fits = fits & ~(twins & torch.ones(m, m, dtype=torch.bool, device=DEV).tril(-1)).any(2)
    fits[:, 0] = True
    holds = ~(_lineage(s) & ~fits[:, None]).any(2)
    count = holds.sum(1)
    ids = torch.arange(m, device=DEV)
    path = torch.where(holds, ids, ids + m).sort(1).values  # the rows that hold, in order, in front
    o["accepted"][:] = torch.where(ids < count[:, None], path, torch.full_like(path, -1))
    o["n_accepted"][:] = count
    o["next_token"][:] = torch.gather(pick, 1, torch.gather(path, 1, count[:, None] - 1))[:, 0]
    o["new_length"][:] = s["length"] + count
    row, to = (ids < count[:, None]).nonzero(as_tuple=True)
    n = s["length"].long()[row]
    from_page, from_place = _slots(s, row, n + path[row, to])
    to_page, to_place = _slots(s, row, n + to)
    for x in (s["k"], s["v"]):
        x[:, to_page, :, to_place] = x[:, from_page, :, from_place]
    return {**o, "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- the framework's calls


def _own(s):
    from yalama_b200 import engine as E
    case, op = s["case"], s["case"]["op"]
    lib, stream = E.lib(), torch.cuda.current_stream().cuda_stream
    if "cache" not in s:  # a program makes these with its buffers
        s["cache"] = E.paged_cache(s["k"].data_ptr(), s["v"].data_ptr(), s["k"].shape[-4], case["page"], case["hkv"])
        s["step"] = E.paged_step(s["row_start"].data_ptr(), s["length"].data_ptr(), s["table"].data_ptr(),
                                 None if s["parent"] is None else s["parent"].data_ptr(), case["seqs"],
                                 s["table"].shape[1], s["rows"], s["max_rows"])
        if op == "attend":
            need = E.paged_attention_workspace(s["cache"], s["step"], case["hq"])
            s["work"] = torch.empty(need, device=DEV, dtype=torch.uint8)
    if op == "append":
        hq, hkv, qkv = case["hq"], case["hkv"], s["qkv"]
        at, norms = qkv.data_ptr(), s["norms"]
        E.check(lib.ylm_k_paged_append(s["cache"], s["step"], at, qkv.stride(0), at + 2 * hq * D, qkv.stride(0),
                                       at + 2 * (hq + hkv) * D, qkv.stride(0), hq,
                                       norms[0].data_ptr() if norms else None, norms[1].data_ptr() if norms else None,
                                       1e-6, s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0],
                                       s["q_out"].data_ptr(), s["q_out"].stride(0), stream), "ylm_k_paged_append")
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if op == "attend":
        E.check(lib.ylm_k_paged_attention(s["cache"], s["step"], s["q"].data_ptr(), s["q"].stride(0), case["hq"],
                                          s["out"].data_ptr(), s["out"].stride(0), s["work"].data_ptr(),
                                          s["work"].numel(), stream), "ylm_k_paged_attention")
        return {"out": s["out"]}
    o = s["out"]
    E.check(lib.ylm_k_paged_accept(s["cache"], s["step"], s["tokens"].data_ptr(), s["picks"].data_ptr(), case["layers"],
                                   s["k"].stride(0), o["accepted"].data_ptr(), o["n_accepted"].data_ptr(),
                                   o["next_token"].data_ptr(), o["new_length"].data_ptr(), stream),
            "ylm_k_paged_accept")
    return {**o, "k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "accept": _plain_accept}[state["case"]["op"]](state)


# ---------------------------------------------------------------- work


def work(case):
    op, hkv = case["op"], case["hkv"]
    n, t = _lengths(case), _rows(case)
    if op == "append":
        heads = case["hq"] + 2 * hkv
        return {"bytes": sum(t) * (4 * D * heads + 2 * D), "flops": sum(t) * 3 * D * heads}
    if op == "attend":
        seen = sum(a * b + (b if case["tree"] else b * (b + 1) // 2) for a, b in zip(n, t))
        return {"bytes": 4 * D * (hkv * sum(a + b for a, b in zip(n, t)) + case["hq"] * sum(t)),
                "flops": 4 * D * case["hq"] * seen}
    moved = sum(_accepted(case)) - case["seqs"] if case["tree"] else 0  # a chain's rows are in place already
    return {"bytes": 8 * D * hkv * case["layers"] * moved + sum(t) * 20 + case["seqs"] * (20 + 4 * max(t)), "flops": sum(t)}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_rows(s):
    """Request by request: its number, its cached tokens, its rows and their parents."""
    case = s["case"]
    at = 0
    for q, (n, t) in enumerate(zip(_lengths(case), _rows(case))):
        p = s["parent"][at:at + t].cpu().tolist() if s["parent"] is not None else list(range(-1, t - 1))
        yield q, n, np.arange(at, at + t), p
        at += t


def _exact_pool(s, kind):
    return s[kind].double()


def _exact_append(s):
    case = s["case"]
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    o = {"q": s["q_out"].double(), "k": _exact_pool(s, "k"), "v": _exact_pool(s, "v")}
    table = s["table"].cpu().numpy()
    for seq, n, rows, parents in _exact_rows(s):
        depth = []
        for p in parents:
            depth.append(0 if p < 0 else depth[p] + 1)
        x = s["qkv"][int(rows[0]):int(rows[-1]) + 1].double()
        heads = x[:, :hq + hkv]
        if s["norms"] is not None:
            w = torch.stack([s["norms"][0]] * hq + [s["norms"][1]] * hkv).double()
            heads = heads / torch.sqrt((heads ** 2).sum(2, keepdim=True) / D + 1e-6) * w
        pos = torch.tensor(depth, device=DEV) + n
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        z = torch.complex(heads[..., :64].contiguous(), heads[..., 64:].contiguous()) * turn
        heads = torch.cat([z.real, z.imag], 2)
        slot = n + np.arange(len(rows))
        to = torch.as_tensor(table[seq, slot // page], device=DEV).long(), torch.as_tensor(slot % page, device=DEV)
        o["q"][int(rows[0]):int(rows[-1]) + 1] = heads[:, :hq]
        o["k"][to[0], :, to[1]] = heads[:, hq:]
        o["v"][to[0], :, to[1]] = x[:, hq + hkv:]
    return o


def _exact_attend(s):
    case = s["case"]
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    group = hq // hkv
    out = s["out"].double()
    for seq, n, rows, parents in _exact_rows(s):
        t, at = len(rows), int(rows[0])
        pages = s["table"][seq, :-(-(n + t) // page)].long()
        see = np.zeros((t, n + t), bool)
        see[:, :n] = True
        for i, p in enumerate(parents):
            if p >= 0:
                see[i, n:] = see[p, n:]
            see[i, n + i] = True
        see = torch.as_tensor(see, device=DEV)
        for h in range(hkv):
            k, v = (s[x][pages, h].reshape(-1, D)[:n + t].double() for x in ("k", "v"))
            for i in range(group):
                x = s["q"][at:at + t, h * group + i].double() @ k.T / math.sqrt(D)
                x[~see] = -math.inf
                out[at:at + t, h * group + i] = torch.softmax(x, 1) @ v
    return {"out": out}


def _exact_accept(s):
    case, page = s["case"], s["case"]["page"]
    seqs, m = case["seqs"], s["max_rows"]
    o = {"accepted": np.full((seqs, m), -1), "n_accepted": np.zeros(seqs, np.int64),
         "next_token": np.zeros(seqs, np.int64), "new_length": np.zeros(seqs, np.int64),
         "k": _exact_pool(s, "k"), "v": _exact_pool(s, "v")}
    token, pick, table = (s[x].cpu().tolist() for x in ("tokens", "picks", "table"))
    for seq, n, rows, parents in _exact_rows(s):
        path = [0]
        while True:
            more = [i for i, p in enumerate(parents) if p == path[-1] and token[rows[i]] == pick[rows[path[-1]]]]
            if not more:
                break
            path.append(more[0])
        o["accepted"][seq, :len(path)] = path
        o["n_accepted"][seq], o["new_length"][seq] = len(path), n + len(path)
        o["next_token"][seq] = pick[rows[path[-1]]]
        for j, i in enumerate(path):  # a path only rises: nothing is overwritten before it has been moved
            a, b = n + i, n + j
            for x in (o["k"], o["v"]):
                x[:, table[seq][b // page], :, b % page] = x[:, table[seq][a // page], :, a % page]
    return o


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "accept": _exact_accept}[case["op"]](s)
