"""Operators of a decoder with sliding-window attention, from training to serving: windowed attention with sinks (dense and
packed sequences, forward and backward), the rotary embedding that writes a paged key-value cache, the attention of the newest
tokens over that cache, and the verification of drafted tokens.

``listed()`` has the fixed cases, ``draw(rng)`` another one of the same ranges.  ``prepare`` makes what a program holds before
the call, ``run`` makes one pass -- the plain formulas in torch, or with ``own`` the framework's operators --, ``work`` counts
the bytes and operations that a pass cannot do without, ``exact`` gives the outputs in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCAB = 32000
THETA = 10000.0


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # prompt processing of one long prompt: grouped heads, the window half of the prompt, four first tokens visible
        {"name": "window_prefill_8192", "kind": "window", "lens": "8192", "packed": False, "H": 32, "Hkv": 8, "window": 4096, "sinks": 4, "dtype": "bf16", "train": False},
        # attention of one training step at sequence length 4096, every head with its own keys
        {"name": "window_train_4096", "kind": "window", "lens": "4096", "packed": False, "H": 32, "Hkv": 32, "window": 1024, "sinks": 4, "dtype": "bf16", "train": True},
        # documents of odd lengths (one of a single token) packed into one training step, odd window, fp16
        {"name": "window_packed_train", "kind": "window", "lens": "1531,1,977,300", "packed": True, "H": 32, "Hkv": 8, "window": 257, "sinks": 3, "dtype": "fp16", "train": True},
        # one user, a short conversation: the smallest call of a server, where latency counts
        {"name": "paged_decode_1x500", "kind": "paged", "B": 1, "n": 1, "lo": 500, "hi": 500, "H": 32, "Hkv": 8, "D": 128, "page": 16, "window": 0, "sinks": 0, "dtype": "bf16"},
        # a full decode batch with a key head for every query head
        {"name": "paged_decode_32x2048", "kind": "paged", "B": 32, "n": 1, "lo": 1100, "hi": 2048, "H": 32, "Hkv": 32, "D": 128, "page": 64, "window": 0, "sinks": 0, "dtype": "bf16"},
        # two very long documents: few rows, so the cache's length has to be split
        {"name": "paged_decode_2x65536", "kind": "paged", "B": 2, "n": 1, "lo": 50001, "hi": 65536, "H": 32, "Hkv": 8, "D": 128, "page": 32, "window": 0, "sinks": 0, "dtype": "bf16"},
        # four drafted tokens and the one before them checked at once, windowed, pages behind the window already given back
        {"name": "paged_check_16x5", "kind": "paged", "B": 16, "n": 5, "lo": 37, "hi": 4001, "H": 32, "Hkv": 8, "D": 64, "page": 32, "window": 1024, "sinks": 4, "dtype": "fp16"},
        # one decode step's rotation and cache update
        {"name": "cache_write_32", "kind": "write", "news": ",".join(["1"] * 32), "before": 1500, "packed": False, "H": 32, "Hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # four prompts of odd lengths written after a prompt prefix that is already there
        {"name": "cache_write_prompts", "kind": "write", "news": "1531,1,2500,64", "before": 33, "packed": True, "H": 32, "Hkv": 8, "D": 128, "page": 16, "dtype": "fp16"},
        # one user, four drafted tokens
        {"name": "verify_1x4", "kind": "verify", "B": 1, "n": 4, "V": VOCAB, "drafts": True, "dtype": "fp32"},
        # a full batch, seven drafted tokens each
        {"name": "verify_64x7", "kind": "verify", "B": 64, "n": 7, "V": VOCAB, "drafts": True, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "paged", "write", "verify"])
    H, Hkv = rng.choice([(32, 32), (32, 8), (16, 2), (8, 1), (6, 3)])
    if kind == "window":
        packed = rng.random() < 0.5
        total = _log_int(rng, 1, 4096)
        lens = [total]
        while packed and len(lens) < 5 and max(lens) > 1:
            longest = lens.pop(lens.index(max(lens)))
            cut = rng.randint(1, longest - 1)
            lens += [cut, longest - cut]
        return {"kind": kind, "lens": ",".join(map(str, lens)), "packed": packed, "H": H, "Hkv": Hkv, "window": _log_int(rng, 1, 4096),
                "sinks": rng.choice([0, 1, 4, 64, 130]), "dtype": rng.choice(["bf16", "fp16"]), "train": rng.random() < 0.6}
    if kind == "paged":
        hi = _log_int(rng, 1, 65536)
        B = max(1, min(_log_int(rng, 1, 64), 131072 // hi))
        n = rng.choice([1, 1, 2, 5, 8])
        return {"kind": kind, "B": B, "n": n, "lo": max(1, hi // rng.randint(1, 50)), "hi": max(hi, n), "H": H, "Hkv": Hkv, "D": rng.choice([64, 128, 128]),
                "page": rng.choice([16, 32, 48, 64, 128]), "window": rng.choice([0, _log_int(rng, 1, 8192)]), "sinks": rng.choice([0, 1, 4, 70]),
                "dtype": rng.choice(["bf16", "fp16"])}
    if kind == "write":
        packed = rng.random() < 0.5
        news = [_log_int(rng, 1, 2000) for _ in range(rng.randint(1, 4))] if packed else [rng.choice([1, 1, 3, 8])] * _log_int(rng, 1, 64)
        return {"kind": kind, "news": ",".join(map(str, news)), "before": rng.randint(0, 1500), "packed": packed, "H": H, "Hkv": Hkv,
                "D": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 48, 64, 128]), "dtype": rng.choice(["bf16", "fp16"])}
    return {"kind": kind, "B": _log_int(rng, 1, 64), "n": rng.randint(1, 8), "V": rng.choice([VOCAB, 50257, 4001, 512]), "drafts": rng.random() < 0.7,
            "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}


def _ints(text):
    return [int(t) for t in text.split(",")]


def _lengths(c):
    """Lengths spread evenly over lo .. hi, the newest tokens included, not in order."""
    B = c["B"]
    lens = [c["hi"] - (c["hi"] - c["lo"]) * i // max(1, B - 1) for i in range(B)]
    return [max(c["n"], lens[(5 * i + 1) % B]) if B % 5 else max(c["n"], lens[i]) for i in range(B)]


# ------------------------------------------------------------------------------------------------ inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=self.g) * std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.g)

    def order(self, n):
        return torch.randperm(n, device="cuda", generator=self.g)


def _place(t):
    """The framework's operators take tensors of its own device; the memory and the values are the same on both."""
    if own:
        import torch_musa_b200  # noqa: F401  (registers the device)

        return t.to("blackwell")
    return t


def _pages(r, lens, page, hidden=lambda b, p: False):
    """A block table of pages in no order, three spare ones in the pool: [sequences, most pages] int32, -1 where there is none."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    ids = r.order(total).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    mask = torch.tensor([[hidden(b, p) for p in range(max(need))] for b in range(len(lens))], device="cuda")
    return table.masked_fill(mask, -1), total


def _inputs(c, seed):
    r, k, dt = _Rand(seed), c["kind"], DTYPES[c["dtype"]]
    if k == "window":
        lens = _ints(c["lens"])
        n = sum(lens)
        shape = (lambda h: (n, h, 128)) if c["packed"] else (lambda h: (1, n, h, 128))
        d = {"q": r.normal(*shape(c["H"]), dtype=dt), "k": r.normal(*shape(c["Hkv"]), dtype=dt), "v": r.normal(*shape(c["Hkv"]), dtype=dt)}
        if c["train"]:
            d["do"] = r.normal(*shape(c["H"]), dtype=dt)
        d["cu"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        return d
    if k == "paged":
        lens, page = _lengths(c), c["page"]

        def given_back(b, p):     # every key of the page lies behind the oldest new token's window and past the sinks
            return bool(c["window"]) and p * page >= c["sinks"] and (p + 1) * page <= lens[b] - c["n"] + 1 - c["window"]

        table, total = _pages(r, lens, page, given_back)
        return {"q": r.normal(c["B"], c["n"], c["H"], c["D"], dtype=dt), "k_pages": r.normal(total, c["Hkv"], page, c["D"], dtype=dt),
                "v_pages": r.normal(total, c["Hkv"], page, c["D"], dtype=dt), "table": table,
                "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    if k == "write":
        news = _ints(c["news"])
        lens = [c["before"] + n for n in news]
        table, total = _pages(r, lens, c["page"])
        t, h, hkv, D = sum(news), c["H"], c["Hkv"], c["D"]
        angle = torch.outer(torch.arange(max(lens), dtype=torch.float64, device="cuda"),
                            THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
        return {"qkv": r.normal(t, h + 2 * hkv, D, dtype=dt), "cos": angle.cos().float(), "sin": angle.sin().float(),
                "k_pages": r.normal(total, hkv, c["page"], D, dtype=dt), "v_pages": r.normal(total, hkv, c["page"], D, dtype=dt), "table": table,
                "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
                "cu": torch.tensor([0] + news, device="cuda").cumsum(0).to(torch.int32)}
    B, n, V = c["B"], c["n"], c["V"]
    base = r.normal(B, n + 1, V, std=2.0)
    d = {"target": torch.softmax(base + r.normal(B, n + 1, V, std=0.5), -1).to(dt), "uniform": r.uniform(B, n + 1)}
    draft = torch.softmax(base[:, :n], -1)
    noise = -torch.log(-torch.log(r.uniform(B, n, V).clamp(1e-7, 1 - 1e-7)))
    d["tokens"] = (draft.log() + noise).argmax(-1) if c["drafts"] else draft.argmax(-1)      # drawn from the draft model, or its first choice
    if c["drafts"]:
        d["draft"] = draft.to(dt)
    return d


def prepare(case, seed):
    s = {"case": case}
    for n, t in _inputs(case, seed).items():
        s[n] = _place(t)
    if case["kind"] == "window" and case["train"]:
        for n in "qkv":
            s[n].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if own:
        return _RUN_OWN[c["kind"]](state, c)
    with torch.no_grad():
        return _RUN_PLAIN[c["kind"]](state, c)


def _own_window(s, c):
    from torch_musa_b200.ops import flash_attn_varlen_func, window_attention

    if c["packed"]:
        longest = max(_ints(c["lens"]))
        out = flash_attn_varlen_func(s["q"], s["k"], s["v"], s["cu"], s["cu"], longest, longest, causal=True, window=c["window"], sinks=c["sinks"])
    else:
        out = window_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"])
    if not c["train"]:
        return [out]
    return [out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])]


def _own_paged(s, c):
    from torch_musa_b200.ops import paged_attention

    return [paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], window=c["window"] or None, sinks=c["sinks"])]


def _split(s, c):
    return s["qkv"].split([c["H"], c["Hkv"], c["Hkv"]], dim=1)


def _own_write(s, c):
    from torch_musa_b200.ops import paged_rope_cache

    q, k, v = _split(s, c)
    out = paged_rope_cache(q, k, v, s["cos"], s["sin"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"] if c["packed"] else None)
    return [out, s["k_pages"], s["v_pages"]]


def _own_verify(s, c):
    from torch_musa_b200.ops import verify_drafts

    return list(verify_drafts(s["target"], s["tokens"], s["uniform"], s.get("draft")))


def _plain_window(s, c):
    q, k, v = (s[n].detach() for n in "qkv")
    shape, dt, T = q.shape, q.dtype, q.shape[-3]
    rows = torch.arange(T, device=q.device)
    seq = (rows[:, None] >= s["cu"][None, 1:-1]).sum(1)
    i, j, first = rows[:, None], rows[None, :], s["cu"][seq].long()[:, None]
    seen = (seq[:, None] == seq[None, :]) & (j <= i) & ((i - j < c["window"]) | (j - first < c["sinks"]))
    G, scale = c["H"] // c["Hkv"], 1.0 / math.sqrt(128)
    heads = lambda t, g: t.reshape(T, c["Hkv"], g, 128).permute(1, 2, 0, 3).float()  # noqa: E731
    qf, kf, vf = heads(q, G), heads(k, 1), heads(v, 1)
    p = (qf @ kf.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    back = lambda t, like: t.permute(2, 0, 1, 3).reshape(like.shape).to(dt)  # noqa: E731
    out = (p @ vf).permute(2, 0, 1, 3).reshape(shape).to(dt)
    if not c["train"]:
        return [out]
    g = heads(s["do"], G)
    ds = g @ vf.transpose(-1, -2)
    ds = ds.sub_((p * ds).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return [out, back(ds @ kf, q), back((ds.transpose(-1, -2) @ qf).sum(1, keepdim=True), k), back((p.transpose(-1, -2) @ g).sum(1, keepdim=True), v)]


def _plain_paged(s, c):
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    B, n, H, D = q.shape
    Hkv, page = s["k_pages"].shape[1:3]
    L = table.shape[1] * page
    gather = lambda pool: pool[table.clamp_min(0)].transpose(1, 2).reshape(B, Hkv, L, D).float()  # noqa: E731
    j = torch.arange(L, device=q.device)
    pos = (lens[:, None] - n + torch.arange(n, device=q.device))[:, :, None]
    seen = (j <= pos) & (table >= 0).repeat_interleave(page, 1)[:, None, :]
    if c["window"]:
        seen = seen & ((pos - j < c["window"]) | (j < c["sinks"]))
    qf = q.float().reshape(B, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    x = (qf @ gather(s["k_pages"]).transpose(-1, -2)).mul_(1.0 / math.sqrt(D))
    x = x.masked_fill_(~seen[:, None, None].expand(B, 1, H // Hkv, n, L).reshape(B, 1, -1, L), float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = (x @ gather(s["v_pages"])) / x.sum(-1, keepdim=True)
    return [o.reshape(B, Hkv, H // Hkv, n, D).permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype)]


def _places(s, page):
    """Position, page and row in the page of every token."""
    t = torch.arange(s["qkv"].shape[0], device=s["qkv"].device)
    cu = s["cu"].long()
    seq = (t[:, None] >= cu[None, 1:-1]).sum(1)
    pos = s["lens"].long()[seq] - (cu[seq + 1] - t)
    return pos, s["table"].long()[seq, pos // page], pos % page


def _plain_write(s, c):
    q, k, v = _split(s, c)
    pos, number, row = _places(s, c["page"])
    cos, sin, half = s["cos"][pos][:, None], s["sin"][pos][:, None], c["D"] // 2

    def rotate(x):
        a, b = x[..., :half].float(), x[..., half:].float()
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(x.dtype)

    s["k_pages"][number, :, row] = rotate(k)
    s["v_pages"][number, :, row] = v
    return [rotate(q), s["k_pages"], s["v_pages"]]


def _plain_verify(s, c):
    p, tokens, u, q = s["target"], s["tokens"], s["uniform"].double(), s.get("draft")
    B, n = tokens.shape
    at = tokens[..., None]
    pt = p[:, :n].gather(2, at).squeeze(2).double()
    qt = q.gather(2, at).squeeze(2).double() if q is not None else torch.ones_like(pt)
    taken = (u[:, :n] * qt < pt).long().cumprod(1).sum(1)
    rows = torch.arange(B, device=p.device)
    w = p[rows, taken].double()
    stop = taken.clamp_max(n - 1)
    if q is not None:
        less = (w - q[rows, stop].double()).clamp_min(0)
    else:
        less = w.scatter(1, tokens[rows, stop][:, None], 0.0)
    w = torch.where((taken < n)[:, None], less, w)
    c = w.cumsum(1)
    last = (c > u[:, n:] * c[:, -1:]).long().argmax(1)
    i = torch.arange(n + 1, device=p.device)
    drafted = torch.cat((tokens, tokens[:, :1]), 1)
    out = torch.where(i < taken[:, None], drafted, torch.where(i == taken[:, None], last[:, None], -1))
    return [taken, out]


_RUN_OWN = {"window": _own_window, "paged": _own_paged, "write": _own_write, "verify": _own_verify}
_RUN_PLAIN = {"window": _plain_window, "paged": _plain_paged, "write": _plain_write, "verify": _plain_verify}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, k = case, case["kind"]
    size = torch.finfo(DTYPES[c["dtype"]]).bits // 8
    if k == "window":
        lens, W, s = _ints(c["lens"]), c["window"], c["sinks"]
        pairs = sum(min(i + 1, W) + min(s, max(0, i + 1 - W)) for n in lens for i in range(n))
        rows, parts = sum(lens) * 128 * size, (4, 4) if c["train"] else (2, 2)      # q, o (do, dq) and k, v (dk, dv)
        return {"bytes": rows * (parts[0] * c["H"] + parts[1] * c["Hkv"]), "flops": (14 if c["train"] else 4) * 128 * pairs * c["H"]}
    if k == "paged":
        n, W = c["n"], c["window"]
        keys = pairs = 0
        for L in _lengths(c):
            first = max(0, L - n + 1 - W) if W else 0
            keys += L - first + min(c["sinks"], first)
            pairs += sum(min(p + 1, W) + min(c["sinks"], max(0, p + 1 - W)) if W else p + 1 for p in range(L - n, L))
        return {"bytes": (2 * keys * c["Hkv"] + 2 * c["B"] * n * c["H"]) * c["D"] * size, "flops": 4 * pairs * c["H"] * c["D"]}
    if k == "write":
        t = sum(_ints(c["news"]))
        return {"bytes": 2 * t * (c["H"] + 2 * c["Hkv"]) * c["D"] * size, "flops": 3 * t * (c["H"] + c["Hkv"]) * c["D"]}
    return {"bytes": c["B"] * (c["V"] * (2 if c["drafts"] else 1) + 2 * c["n"]) * size, "flops": 3 * c["B"] * c["V"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    with torch.no_grad():
        d = _inputs(case, seed)
        return _EXACT[case["kind"]](d, case)


def _exact_window(d, c):
    """Sequence by sequence and head by head, the gradients by the chain rule."""
    lens, W, s = _ints(c["lens"]), c["window"], c["sinks"]
    flat = {n: t.reshape(-1, t.shape[-2], 128).double() for n, t in d.items() if n != "cu"}
    out = {n: torch.zeros_like(flat[m]) for n, m in (("o", "q"), ("q", "q"), ("k", "k"), ("v", "v"))}
    G, at = c["H"] // c["Hkv"], 0
    for n in lens:
        here = slice(at, at + n)
        at += n
        away = torch.arange(n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None, :]
        bias = torch.zeros(n, n, dtype=torch.float64, device="cuda")
        far = away >= W
        far[:, :s] = False
        bias[far | (away < 0)] = -math.inf
        for h in range(c["H"]):
            q, k, v = flat["q"][here, h], flat["k"][here, h // G], flat["v"][here, h // G]
            p = torch.softmax(q @ k.T / math.sqrt(128) + bias, dim=1)
            o = p @ v
            out["o"][here, h] = o
            if c["train"]:
                g = flat["do"][here, h]
                ds = p * (g @ v.T - (g * o).sum(1, keepdim=True)) / math.sqrt(128)
                out["q"][here, h] = ds @ k
                out["k"][here, h // G] += ds.T @ q
                out["v"][here, h // G] += p.T @ g
    shaped = [out["o"].reshape(d["q"].shape)]
    return shaped + [out[n].reshape(d[n].shape) for n in "qkv"] if c["train"] else shaped


def _exact_paged(d, c):
    """Sequence by sequence over the keys that its newest tokens see."""
    out = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    G, n = c["H"] // c["Hkv"], c["n"]
    for b, L in enumerate(_lengths(c)):
        j = torch.arange(L, device="cuda")
        number, row = d["table"][b].long()[j // c["page"]], j % c["page"]
        k = d["k_pages"][number, :, row].double().transpose(0, 1)             # [Hkv, L, D]; a hidden page's keys are never chosen below
        v = d["v_pages"][number, :, row].double().transpose(0, 1)
        for t in range(n):
            p = L - n + t
            seen = (j <= p) if not c["window"] else (j <= p) & ((j > p - c["window"]) | (j < c["sinks"]))
            q = d["q"][b, t].double().reshape(c["Hkv"], G, -1)
            w = torch.softmax(q @ k[:, seen].transpose(1, 2) / math.sqrt(c["D"]), dim=-1)
            out[b, t] = (w @ v[:, seen]).reshape(c["H"], -1)
    return [out]


def _exact_write(d, c):
    q, k, v = (t.double() for t in _split(d, c))
    pools = [d["k_pages"].double(), d["v_pages"].double()]
    half, t, turned = c["D"] // 2, 0, torch.empty_like(q)
    for b, n in enumerate(_ints(c["news"])):
        pos = torch.arange(c["before"], c["before"] + n, device="cuda")
        number, row = d["table"][b].long()[pos // c["page"]], pos % c["page"]
        z = torch.complex(d["cos"][pos].double(), d["sin"][pos].double())[:, None]
        turn = lambda x: torch.cat(((y := torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * z).real, y.imag), -1)  # noqa: E731
        turned[t:t + n] = turn(q[t:t + n])
        pools[0][number, :, row] = turn(k[t:t + n])
        pools[1][number, :, row] = v[t:t + n]
        t += n
    return [turned, *pools]


def _exact_verify(d, c):
    """Whole numbers, found one sequence and one token at a time."""
    taken, rows = [], []
    for b in range(c["B"]):
        p, u, x = d["target"][b].double().cpu(), d["uniform"][b].double().tolist(), d["tokens"][b].tolist()
        q = d["draft"][b].double().cpu() if c["drafts"] else None
        r = 0
        while r < c["n"] and u[r] * (float(q[r, x[r]]) if c["drafts"] else 1.0) < float(p[r, x[r]]):
            r += 1
        w = p[r].clone()
        if r < c["n"]:
            if c["drafts"]:
                w = (w - q[r]).clamp_min(0)
            else:
                w[x[r]] = 0
        total = w.cumsum(0)
        token = int(torch.searchsorted(total, torch.tensor([u[c["n"]] * float(total[-1])], dtype=torch.float64), right=True))
        taken.append(r)
        rows.append(x[:r] + [token] + [-1] * (c["n"] - r))
    return [torch.tensor(taken), torch.tensor(rows)]


_EXACT = {"window": _exact_window, "paged": _exact_paged, "write": _exact_write, "verify": _exact_verify}
