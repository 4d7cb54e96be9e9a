"""The operators of a long request on a fixed key/value budget, and the cases they are measured on.

- store:    FP16 key and value rows into an 8-bit cache with one power-of-two scale per block of tokens and head
- attend:   attention of the last tokens over that cache, with the attention weight accumulated per slot
- evict:    the slots of largest accumulated weight kept, in order, in another cache
- logprobs: log probability of a given token, entropy and the most likely alternatives of rows of FP16 logits

``run`` computes them in elementary torch operations, or with the framework's kernels where ``own`` is true.
"""
import math

import numpy as np
import torch

own = False

D = 128                                    # head dimension
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}  # largest magnitude of a code
DEV = "cuda"


def listed():
    return [
        # one decode step's key and value (Llama-3.1-8B heads) appended inside a block: latency
        {"name": "store 1 e4m3", "op": "store", "fmt": "e4m3", "hkv": 8, "block": 32, "t": 1, "slot": 2611},
        # the prompt of the default benchmark, one layer, into an empty cache
        {"name": "store 2048 e4m3", "op": "store", "fmt": "e4m3", "hkv": 8, "block": 64, "t": 2048, "slot": 0},
        # a later, odd piece of a prompt behind cached tokens (Qwen2.5-7B heads)
        {"name": "store 777 int8", "op": "store", "fmt": "int8", "hkv": 4, "block": 16, "t": 777, "slot": 5003},
        # a decode step early in a chat: latency
        {"name": "attend 1x611 e4m3", "op": "attend", "fmt": "e4m3", "hq": 24, "hkv": 8, "block": 32, "t": 1,
         "n": 611, "acc": False, "mask": False},
        # a decode step behind a long prompt, weights kept for a later eviction (Qwen2.5-7B heads)
        {"name": "attend 1x8200 int8", "op": "attend", "fmt": "int8", "hq": 28, "hkv": 4, "block": 64, "t": 1,
         "n": 8200, "acc": True, "mask": False},
        # a decode step at the end of the longest context (Llama-3.1-8B heads)
        {"name": "attend 1x131071 e4m3", "op": "attend", "fmt": "e4m3", "hq": 32, "hkv": 8, "block": 128, "t": 1,
         "n": 131071, "acc": True, "mask": False},
        # eight drafted tokens verified at once, some slots hidden (Llama-3.1-70B heads)
        {"name": "attend 8x4099 e4m3", "op": "attend", "fmt": "e4m3", "hq": 64, "hkv": 8, "block": 64, "t": 8,
         "n": 4099, "acc": True, "mask": True},
        # a small budget halved
        {"name": "evict 2100 int8", "op": "evict", "fmt": "int8", "hkv": 8, "block": 16, "n": 2100, "n_keep": 1024,
         "n_sink": 4, "n_recent": 128},
        # a long context cut to the slots that are looked at
        {"name": "evict 65536 e4m3", "op": "evict", "fmt": "e4m3", "hkv": 8, "block": 64, "n": 65536,
         "n_keep": 40000, "n_sink": 4, "n_recent": 4096},
        # the step of a service that returns `logprobs`: one row, the most alternatives such a request may ask for
        {"name": "logprobs 1x128256", "op": "logprobs", "rows": 1, "vocab": 128256, "n_top": 20, "mask": False},
        # drafted tokens scored, special tokens masked, a small vocabulary (Mistral-7B)
        {"name": "logprobs 37x32768", "op": "logprobs", "rows": 37, "vocab": 32768, "n_top": 5, "mask": True},
        # a piece of a prompt scored (Qwen3-0.6B's vocabulary)
        {"name": "logprobs 600x151936", "op": "logprobs", "rows": 600, "vocab": 151936, "n_top": 8, "mask": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "evict", "logprobs"])
    fmt, block = rng.choice(["e4m3", "int8"]), rng.choice([16, 32, 64, 128])
    if op == "store":
        return {"op": op, "fmt": fmt, "hkv": rng.choice([1, 2, 4, 8]), "block": block, "t": _log(rng, 1, 4096),
                "slot": rng.choice([0, _log(rng, 1, 20000)])}
    if op == "attend":
        hq, hkv = rng.choice([(16, 8), (24, 8), (28, 4), (32, 8), (64, 8), (8, 8), (8, 1), (14, 2)])
        t = rng.choice([1, 1, rng.randint(2, 16)])
        n = _log(rng, max(t, 16), 131071 if t == 1 and hq <= 32 else 16384)
        return {"op": op, "fmt": fmt, "hq": hq, "hkv": hkv, "block": block, "t": t, "n": n,
                "acc": rng.random() < 0.6, "mask": rng.random() < 0.4}
    if op == "evict":
        n = _log(rng, 200, 65536)
        keep = max(64, min(n - 1, int(n * rng.uniform(0.2, 0.6))))
        return {"op": op, "fmt": fmt, "hkv": rng.choice([1, 2, 4, 8]), "block": block, "n": n, "n_keep": keep,
                "n_sink": rng.randint(0, 8), "n_recent": rng.randint(0, keep // 2)}
    return {"op": op, "rows": _log(rng, 1, 500), "vocab": rng.choice([32768, 128256, 151936, _log(rng, 2000, 150000)]),
            "n_top": rng.randint(0, 20), "mask": rng.random() < 0.4}


# ---------------------------------------------------------------- inputs


def _rows(g, t, hkv, kind):
    """[t, hkv, 128] FP16 keys (a few strong channels, as rotated keys have) or values (weak first tokens)."""
    x = torch.randn(t, hkv, D, generator=g, device=DEV)
    gain = torch.exp(0.5 * torch.randn(hkv, D, generator=g, device=DEV))
    if kind == "k":
        x = x * gain
    else:
        x = x * 0.4
        x[:4] *= 0.02
    return x.half()


def _scale_of(amax, fmt):
    """The smallest power of two s with amax <= CODE_MAX s; 0 for amax = 0 (elementwise)."""
    m, e = torch.frexp(amax)
    top = CODE_MAX[fmt]
    mt, et = math.frexp(top)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - et + (m > mt).int()), torch.zeros_like(amax))


def _codes(x, s, fmt):
    """FP32 values x over scales s, as codes (uint8)."""
    y = x / torch.where(s > 0, s, torch.ones_like(s))
    if fmt == "e4m3":
        return y.to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.round(y).to(torch.int8).view(torch.uint8)


def _numbers(codes, fmt):
    """The numbers that codes stand for, in units of their scale: a view, no copy."""
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8)


def _cache(g, case, n, cap):
    """An 8-bit cache with slots [0, n) filled, as separate stores would have left it; the slots behind hold anything
    (but no NaN where the whole cache is an output)."""
    hkv, block, fmt = case["hkv"], case["block"], case["fmt"]
    nb = -(-cap // block)
    c = {"cap": cap}
    for kind in ("k", "v"):
        x = _rows(g, n, hkv, kind).float().permute(1, 0, 2)
        x = torch.nn.functional.pad(x, (0, 0, 0, nb * block - n)).reshape(hkv, nb, block, D)
        s = _scale_of(x.abs().amax((2, 3)), fmt)
        c[kind] = _codes(x, s[:, :, None, None], fmt).reshape(hkv, nb * block, D)[:, :cap].contiguous()
        c[kind + "_scale"] = s.contiguous()
        c[kind][:, n:] = torch.randint(0, 256, (hkv, cap - n, D), generator=g, device=DEV, dtype=torch.uint8)
        if case["op"] == "store":
            c[kind][:, n:] &= 0xF7
    return c


def _weights(g, hkv, cap, n):
    """Accumulated attention weight as many steps leave it: heavy-tailed, and exactly 0 for some slots."""
    a = torch.exp(2.5 * torch.randn(hkv, cap, generator=g, device=DEV) - 4)
    a[torch.rand(hkv, cap, generator=g, device=DEV) < 0.05] = 0
    a[:, n:] = 0
    return a


def _pack_bits(hidden):
    """Bools as the framework's mask words: bit i & 31 of word i >> 5 hides i."""
    n = hidden.numel()
    b = torch.nn.functional.pad(hidden, (0, -n % 32)).reshape(-1, 32).long()
    w = (b << torch.arange(32, device=DEV)).sum(1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "store":
        n = case["slot"] + case["t"]
        s["cache"] = _cache(g, case, case["slot"], n + 100)
        # the new rows lie in the rows of a fused projection, as the model path has them
        qkv = torch.randn(case["t"], 4 * case["hkv"], D, generator=g, device=DEV).half()
        qkv[:, 2 * case["hkv"]:3 * case["hkv"]] = _rows(g, case["t"], case["hkv"], "k")
        qkv[:, 3 * case["hkv"]:] = _rows(g, case["t"], case["hkv"], "v")
        s["k_new"], s["v_new"] = qkv[:, 2 * case["hkv"]:3 * case["hkv"]], qkv[:, 3 * case["hkv"]:]
    elif op == "attend":
        n, cap = case["n"], case["n"] + 130
        s["cache"] = _cache(g, case, n, cap)
        s["q"] = torch.randn(case["t"], case["hq"], D, generator=g, device=DEV).half()
        s["out"] = torch.empty(case["t"], case["hq"] * D, device=DEV, dtype=torch.float16)
        s["acc"] = _weights(g, case["hkv"], cap, n) if case["acc"] else None
        s["bits"] = _pack_bits(torch.rand(cap, generator=g, device=DEV) < 0.1) if case["mask"] else None
    elif op == "evict":
        n, keep, hkv, block = case["n"], case["n_keep"], case["hkv"], case["block"]
        s["cache"] = _cache(g, case, n, n + 70)
        s["acc"] = _weights(g, hkv, n + 70, n)
        cap, nb = keep + 90, -(-(keep + 90) // block)
        s["dst"] = {"cap": cap, "k": torch.zeros(hkv, cap, D, device=DEV, dtype=torch.uint8),
                    "v": torch.zeros(hkv, cap, D, device=DEV, dtype=torch.uint8),
                    "k_scale": torch.zeros(hkv, nb, device=DEV), "v_scale": torch.zeros(hkv, nb, device=DEV)}
        s["dst_acc"] = torch.zeros(hkv, cap, device=DEV)
        s["kept"] = torch.zeros(hkv, keep, device=DEV, dtype=torch.int32)
    else:
        rows, vocab, k = case["rows"], case["vocab"], case["n_top"]
        x = torch.randn(rows, vocab, generator=g, device=DEV)
        # rows from nearly uniform to nearly certain
        x *= 1.5 + 1.5 * torch.rand(rows, 1, generator=g, device=DEV)
        x[torch.arange(rows, device=DEV), torch.randint(0, vocab, (rows,), generator=g, device=DEV)] += \
            16 * torch.rand(rows, generator=g, device=DEV)
        s["logits"] = x.half()
        s["ids"] = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        s["ids"][::2] = s["logits"][::2].argmax(1)
        s["bits"] = _pack_bits(torch.rand(vocab, generator=g, device=DEV) < 0.01) if case["mask"] else None
        s["out"] = {"logprob": torch.empty(rows, device=DEV), "entropy": torch.empty(rows, device=DEV),
                    "top_ids": torch.empty(rows, k, device=DEV, dtype=torch.int64),
                    "top_logprobs": torch.empty(rows, k, device=DEV)}
    return s


# ---------------------------------------------------------------- plain forms


def _values(c, name, n, case):
    """Slots [0, n) of a cache's keys or values, in 32 bits."""
    x = _numbers(c[name][:, :n].contiguous(), case["fmt"]).float()
    return x * c[name + "_scale"].repeat_interleave(case["block"], 1)[:, :n, None]


def _hidden(bits, n):
    """Mask words as bools."""
    i = torch.arange(n, device=DEV)
    return (bits[i >> 5] >> (i & 31).int()) & 1 != 0


def _plain_store(s):
    case, c = s["case"], s["cache"]
    t, slot, block, fmt = case["t"], case["slot"], case["block"], case["fmt"]
    b0, b1 = slot // block, (slot + t - 1) // block
    first = b0 * block
    nb, held = b1 - b0 + 1, slot - first
    for kind in ("k", "v"):
        x = s[kind + "_new"].float().permute(1, 0, 2)
        x = torch.nn.functional.pad(x, (0, 0, held, nb * block - held - t)).reshape(-1, nb, block, D)
        new = _scale_of(x.abs().amax((2, 3)), fmt)
        if held:
            old = c[kind + "_scale"][:, b0].clone()
            new[:, 0] = torch.maximum(new[:, 0], old)
            before = _numbers(c[kind][:, first:slot].contiguous(), fmt).float() * old[:, None, None]
            c[kind][:, first:slot] = _codes(before, new[:, :1, None], fmt)
        codes = _codes(x, new[:, :, None, None], fmt).reshape(-1, nb * block, D)
        c[kind][:, slot:slot + t] = codes[:, held:held + t]
        c[kind + "_scale"][:, b0:b1 + 1] = new
    return _cache_out(c, fmt)


def _plain_attend(s):
    case, c = s["case"], s["cache"]
    t, n, hq, hkv = case["t"], case["n"], case["hq"], case["hkv"]
    k, v = _values(c, "k", n, case), _values(c, "v", n, case)
    q = s["q"].float().reshape(t, hkv, hq // hkv, D).permute(1, 0, 2, 3).reshape(hkv, -1, D)
    x = (q @ k.transpose(1, 2)) * (1 / math.sqrt(D))
    x = x.reshape(hkv, t, hq // hkv, n)
    slot = torch.arange(n, device=DEV)
    hide = slot > torch.arange(n - t, n, device=DEV)[:, None]
    if s["bits"] is not None:
        hide = hide | _hidden(s["bits"], n)
    x = x.masked_fill(hide[None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z > 0, z, torch.ones_like(z))).reshape(hkv, -1, n)
    o = (p @ v).reshape(hkv, t, -1, D).permute(1, 0, 2, 3).reshape(t, hq * D).half()
    if s["acc"] is not None:
        s["acc"][:, :n] += p.sum(1)
    return {"out": o, "acc": s["acc"]}


def _plain_evict(s):
    case, c, d, acc = s["case"], s["cache"], s["dst"], s["acc"]
    n, keep, block, fmt = case["n"], case["n_keep"], case["block"], case["fmt"]
    key = acc[:, :n].clone()
    key[:, :case["n_sink"]] = math.inf
    key[:, n - case["n_recent"]:] = math.inf
    kept = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :keep].sort(1).values
    nb = -(-keep // block)
    for kind in ("k", "v"):
        old = torch.gather(c[kind + "_scale"], 1, kept // block)
        new = torch.nn.functional.pad(old, (0, nb * block - keep)).reshape(-1, nb, block).amax(2)
        x = _numbers(torch.gather(c[kind], 1, kept[:, :, None].expand(-1, -1, D)), fmt).float() * old[:, :, None]
        d[kind][:, :keep] = _codes(x, new.repeat_interleave(block, 1)[:, :keep, None], fmt)
        d[kind + "_scale"][:, :nb] = new
    s["dst_acc"].zero_()
    s["dst_acc"][:, :keep] = torch.gather(acc, 1, kept)
    s["kept"].copy_(kept)
    return {"kept": s["kept"], "acc": s["dst_acc"], **_cache_out(d, fmt)}


def _plain_logprobs(s):
    case = s["case"]
    x = s["logits"].float()
    if s["bits"] is not None:
        x = x.masked_fill(_hidden(s["bits"], case["vocab"]), -math.inf)
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    o = {"logprob": (d.gather(1, s["ids"][:, None]) - log_z)[:, 0],
         "entropy": (log_z - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1, keepdim=True) / z)[:, 0]}
    if case["n_top"]:
        top = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :case["n_top"]]
        o["top_ids"], o["top_logprobs"] = top, d.gather(1, top) - log_z
    return o


def _cache_out(c, fmt):
    """A cache's buffers: what the codes stand for, in units of the scale of their block, and the scales."""
    return {"k": _numbers(c["k"], fmt), "v": _numbers(c["v"], fmt), "k_scale": c["k_scale"], "v_scale": c["v_scale"]}


# ---------------------------------------------------------------- the framework's calls


def _address(x):
    return None if x is None else x.data_ptr()


def _handle(E, c, case):
    return E.kv8_cache(c["k"].data_ptr(), c["v"].data_ptr(), c["k_scale"].data_ptr(), c["v_scale"].data_ptr(),
                       case["fmt"], case["block"], c["cap"], case["hkv"])


def _own(s):
    from yalama_b200 import engine as E
    case, op = s["case"], s["case"]["op"]
    lib, stream = E.lib(), torch.cuda.current_stream().cuda_stream
    if op != "logprobs" and "handle" not in s:  # a program makes these with its buffers
        s["handle"] = _handle(E, s["cache"], case)
        if op == "evict":
            s["dst_handle"] = _handle(E, s["dst"], case)
        if op == "attend":
            need = E.kv8_attention_workspace(s["handle"], case["hq"], case["t"], case["n"], case["acc"])
            s["work"] = torch.empty(need, device=DEV, dtype=torch.uint8)
    if op == "store":
        E.check(lib.ylm_k_kv8_store(s["handle"], s["k_new"].data_ptr(), s["k_new"].stride(0), s["v_new"].data_ptr(),
                                    s["v_new"].stride(0), case["t"], case["slot"], stream), "ylm_k_kv8_store")
        return _cache_out(s["cache"], case["fmt"])
    if op == "attend":
        E.check(lib.ylm_k_kv8_attention(s["handle"], s["q"].data_ptr(), s["q"].stride(0), case["hq"], case["t"],
                                        case["n"], _address(s["bits"]), _address(s["acc"]), s["out"].data_ptr(),
                                        s["out"].stride(0), s["work"].data_ptr(), s["work"].numel(), stream),
                "ylm_k_kv8_attention")
        return {"out": s["out"], "acc": s["acc"]}
    if op == "evict":
        E.check(lib.ylm_k_kv8_evict(s["handle"], s["dst_handle"], s["acc"].data_ptr(), s["dst_acc"].data_ptr(),
                                    case["n"], case["n_keep"], case["n_sink"], case["n_recent"],
                                    s["kept"].data_ptr(), stream), "ylm_k_kv8_evict")
        return {"kept": s["kept"], "acc": s["dst_acc"], **_cache_out(s["dst"], case["fmt"])}
    o = s["out"]
    E.check(lib.ylm_k_logprobs(s["logits"].data_ptr(), s["logits"].stride(0), case["rows"], case["vocab"],
                               s["ids"].data_ptr(), _address(s["bits"]), case["n_top"], o["logprob"].data_ptr(),
                               o["entropy"].data_ptr(), o["top_ids"].data_ptr(), o["top_logprobs"].data_ptr(),
                               stream), "ylm_k_logprobs")
    return o if case["n_top"] else {"logprob": o["logprob"], "entropy": o["entropy"]}


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attend": _plain_attend, "evict": _plain_evict,
            "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# ---------------------------------------------------------------- work


def work(case):
    op = case["op"]
    if op == "store":
        t, hkv = case["t"], case["hkv"]
        return {"bytes": 2 * t * hkv * (3 * D) + 8 * hkv * (-(-t // case["block"])), "flops": 4 * t * hkv * D}
    if op == "attend":
        t, n, hq, hkv = case["t"], case["n"], case["hq"], case["hkv"]
        b = 2 * n * hkv * D + 8 * hkv * (-(-n // case["block"])) + 4 * t * hq * D
        b += (8 * n * hkv if case["acc"] else 0) + (n // 8 if case["mask"] else 0)
        return {"bytes": b, "flops": 4 * n * t * hq * D}
    if op == "evict":
        n, keep, hkv = case["n"], case["n_keep"], case["hkv"]
        return {"bytes": hkv * (4 * n + keep * (4 * D + 8) + 8 * (-(-n // case["block"]) + -(-keep // case["block"]))),
                "flops": 2 * keep * hkv * D}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (2 * vocab + 16 + 12 * case["n_top"]), "flops": 5 * rows * vocab}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_codes(c, kind, case):
    """Codes as numbers in 64 bits, decoded from their bits."""
    b = c[kind].cpu().numpy()
    if case["fmt"] == "int8":
        return b.view(np.int8).astype(np.float64)
    e, m = (b >> 3) & 15, (b & 7).astype(np.float64)
    mag = np.where(e > 0, (1 + m / 8) * np.exp2(e.astype(np.float64) - 7), m / 8 * 2.0 ** -6)
    mag = np.where((b & 127) == 127, np.nan, mag)
    return np.where(b & 128, -mag, mag)


def _exact_scale(amax, fmt):
    """2^ceil(log2(amax / CODE_MAX)), with the exponent put right where the logarithm's rounding moved it."""
    a = np.asarray(amax, np.float64)
    e = np.ceil(np.log2(np.where(a > 0, a, 1) / CODE_MAX[fmt]))
    e = np.where(a > CODE_MAX[fmt] * np.exp2(e), e + 1, e)
    e = np.where(a <= CODE_MAX[fmt] * np.exp2(e - 1), e - 1, e)
    return np.where(a > 0, np.exp2(e), 0.0)


def _exact_store(s):
    case, c = s["case"], s["cache"]
    t, slot, block, fmt = case["t"], case["slot"], case["block"], case["fmt"]
    o = {}
    for kind in ("k", "v"):
        codes, scale = _exact_codes(c, kind, case), c[kind + "_scale"].cpu().numpy().astype(np.float64)
        new = s[kind + "_new"].cpu().numpy().astype(np.float64).transpose(1, 0, 2)
        for b in range(slot // block, (slot + t - 1) // block + 1):
            lo, hi = max(slot, b * block), min(slot + t, (b + 1) * block)
            x = new[:, lo - slot:hi - slot]
            want = _exact_scale(np.abs(x).max((1, 2)), fmt)
            if lo > b * block:
                want = np.maximum(want, scale[:, b])
                codes[:, b * block:lo] *= (scale[:, b] / np.where(want > 0, want, 1))[:, None, None]
            codes[:, lo:hi] = x / np.where(want > 0, want, 1)[:, None, None]
            scale[:, b] = want
        # integer codes are whole numbers and have no value between them
        o[kind], o[kind + "_scale"] = (None if fmt == "int8" else codes), scale
    return o


def _exact_attend(s):
    case, c = s["case"], s["cache"]
    t, n, hq, hkv = case["t"], case["n"], case["hq"], case["hkv"]
    group = hq // hkv
    bits = None if s["bits"] is None else \
        np.unpackbits(s["bits"].cpu().numpy().view(np.uint8), bitorder="little")[:n].astype(bool)
    out = torch.zeros(t, hq, D, dtype=torch.float64)
    acc = None if s["acc"] is None else s["acc"].double().cpu()
    slot = torch.arange(n, device=DEV)
    number = torch.from_numpy(_exact_codes({"x": torch.arange(256, dtype=torch.uint8)}, "x", case)).to(DEV)
    for h in range(hkv):
        k, v = (number[c[kind][h, :n].long()] *
                c[kind + "_scale"][h].double()[slot // case["block"]][:, None] for kind in ("k", "v"))
        for i in range(t):
            see = slot <= n - t + i
            if bits is not None:
                see &= ~torch.from_numpy(bits).to(DEV)
            if not bool(see.any()):
                continue
            x = s["q"][i, h * group:(h + 1) * group].double() @ k[see].T / math.sqrt(D)
            p = torch.softmax(x, 1)
            out[i, h * group:(h + 1) * group] = (p @ v[see]).cpu()
            if acc is not None:
                acc[h, :n][see.cpu()] += p.sum(0).cpu()
    return {"out": out.reshape(t, hq * D), "acc": acc}


def _exact_evict(s):
    case, c = s["case"], s["cache"]
    n, keep, block, hkv = case["n"], case["n_keep"], case["block"], case["hkv"]
    acc = s["acc"].cpu().numpy().astype(np.float64)
    kept = np.empty((hkv, keep), np.int64)
    inner = np.arange(case["n_sink"], n - case["n_recent"])
    held = np.concatenate([np.arange(case["n_sink"]), np.arange(n - case["n_recent"], n)])
    for h in range(hkv):
        best = inner[np.lexsort((inner, -acc[h, inner]))][:keep - held.size]
        kept[h] = np.sort(np.concatenate([held, best]))
    o = {"kept": kept, "acc": np.zeros((hkv, s["dst"]["cap"]))}
    o["acc"][:, :keep] = np.take_along_axis(acc, kept, 1)
    for kind in ("k", "v"):
        codes, scale = _exact_codes(c, kind, case), c[kind + "_scale"].cpu().numpy().astype(np.float64)
        new = np.zeros(s["dst"][kind + "_scale"].shape)
        num = np.zeros((hkv, s["dst"]["cap"], D))
        for b in range(-(-keep // block)):
            at = kept[:, b * block:min(keep, (b + 1) * block)]
            old = np.take_along_axis(scale, at // block, 1)
            new[:, b] = old.max(1)
            ratio = old / np.where(new[:, b] > 0, new[:, b], 1)[:, None]
            num[:, b * block:b * block + at.shape[1]] = np.take_along_axis(codes, at[:, :, None], 1) * ratio[:, :, None]
        o[kind], o[kind + "_scale"] = (None if case["fmt"] == "int8" else num), new
    return o


def _exact_logprobs(s):
    case = s["case"]
    rows, vocab, k = case["rows"], case["vocab"], case["n_top"]
    seen = np.ones(vocab, bool)
    if s["bits"] is not None:
        seen = ~np.unpackbits(s["bits"].cpu().numpy().view(np.uint8), bitorder="little")[:vocab].astype(bool)
    open_ids = torch.from_numpy(np.nonzero(seen)[0]).to(DEV)
    o = {"logprob": np.empty(rows), "entropy": np.empty(rows)}
    if k:
        o["top_ids"], o["top_logprobs"] = np.empty((rows, k), np.int64), np.empty((rows, k))
    for r in range(rows):
        x = s["logits"][r].double()
        lp = torch.log_softmax(x[open_ids], 0)
        whole = torch.full((vocab,), -math.inf, dtype=torch.float64, device=DEV)
        whole[open_ids] = lp
        o["logprob"][r] = whole[s["ids"][r]].item()
        o["entropy"][r] = -(lp.exp() * lp).sum().item()
        if k:
            # the k best by value and then by id, from the few that reach the k-th value
            lowest = torch.topk(x[open_ids], k).values[-1]
            few = open_ids[x[open_ids] >= lowest].cpu().numpy()
            vals = x.cpu().numpy()[few]
            best = few[np.lexsort((few, -vals))][:k]
            o["top_ids"][r], o["top_logprobs"][r] = best, whole.cpu().numpy()[best]
    return o


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "evict": _exact_evict,
            "logprobs": _exact_logprobs}[case["op"]](s)
