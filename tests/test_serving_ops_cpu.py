"""Windowed attention, the paged cache and the verification of drafts off the device: the plain formulation against loops in 64
bits, refusals, and the paged decoder against the model run from scratch."""
import ctypes
import math
import os

import pytest
import torch

import torch_musa_b200
from torch_musa_b200 import ops
from torch_musa_b200.models import Llama, PagedLlamaDecoder, llama_tiny_config
from torch_musa_b200.models.decode import LlamaDecoder

U = 2.0 ** -24      # half a step of float32


def loop_attention(q, k, v, seen):
    """q [n, D], k / v [L, D], seen [n, L]; rows that see nothing are zero."""
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    for i in range(q.shape[0]):
        at = torch.nonzero(seen[i]).flatten()
        if len(at):
            out[i] = torch.softmax(k[at].double() @ q[i].double() / math.sqrt(q.shape[1]), 0) @ v[at].double()
    return out


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (100, 1)])
def test_window_attention_and_its_packed_form(window, sinks):
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(1, 20, 4, 16, generator=g), torch.randn(1, 20, 2, 16, generator=g), torch.randn(1, 20, 2, 16, generator=g)
    out = ops.window_attention(q, k, v, window, sinks)
    i, j = torch.arange(20)[:, None], torch.arange(20)[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    for h in range(4):
        want = loop_attention(q[0, :, h], k[0, :, h // 2], v[0, :, h // 2], seen)
        # 32-bit sums of 16 products, an exponential and 20 weights: under 64 half steps of values below 8
        assert float((out[0, :, h].double() - want).abs().max()) <= 64 * U * 8
    cu = torch.tensor([0, 0, 7, 18], dtype=torch.int32)
    packed = ops.flash_attn_varlen_func(q[0], k[0], v[0], cu, cu, 11, 11, causal=True, window=window, sinks=sinks)
    for a, b in ((0, 7), (7, 18)):
        assert torch.allclose(packed[a:b], ops.window_attention(q[:, a:b], k[:, a:b], v[:, a:b], window, sinks)[0], rtol=0, atol=64 * U * 8)
    assert bool((packed[18:] == 0).all())


def test_window_refusals():
    q = torch.zeros(1, 4, 2, 16)
    for bad in (lambda: ops.window_attention(q, q, q, 0), lambda: ops.window_attention(q, q, q, 4, -1),
                lambda: ops.window_attention(q, q[:, :, :0], q[:, :, :0], 4), lambda: ops.window_attention(q, q.expand(2, -1, -1, -1), q, 4),
                lambda: ops.window_attention(q[0], q[0], q[0], 4),
                lambda: ops.flash_attn_varlen_func(q[0], q[0], q[0], torch.tensor([0, 4]), torch.tensor([0, 4]), 4, 4, window=2),
                lambda: ops.flash_attn_varlen_func(q[0], q[0], q[0], torch.tensor([0, 4]), torch.tensor([0, 4]), 4, 4, causal=True, window=-1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="PagedLlamaDecoder"):
        LlamaDecoder(Llama(llama_tiny_config(window=8)), 1, 16)


def paged_case(seed, lens, n, H=4, Hkv=2, D=16, page=16, pages=12):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    width = max(1, max(-(-x // page) for x in lens))
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, x in enumerate(lens):
        need = -(-x // page)
        table[b, :need] = ids[at:at + need]
        at += need
    pool = lambda: torch.randn(pages, Hkv, page, D, generator=g)  # noqa: E731
    return torch.randn(len(lens), n, H, D, generator=g), pool(), pool(), table, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.parametrize("n,window,sinks", [(1, None, 0), (3, None, 0), (3, 5, 0), (2, 4, 17), (1, 1, 1)])
def test_paged_attention(n, window, sinks):
    q, kp, vp, table, lens = paged_case(1, [1, 0, 33, 16, 50], n)
    out = ops.paged_attention(q, kp, vp, table, lens, window, sinks)
    for b, L in enumerate(lens.tolist()):
        number, row = table[b].long()[torch.arange(L) // 16], torch.arange(L) % 16
        pos, j = L - n + torch.arange(n)[:, None], torch.arange(L)[None]
        seen = j <= pos if window is None else (j <= pos) & ((pos - j < window) | (j < sinks))
        for h in range(4):
            want = loop_attention(q[b, :, h], kp[number, h // 2, row], vp[number, h // 2, row], seen)
            assert float((out[b, :, h].double() - want).abs().max()) <= 64 * U * 8


def test_paged_attention_reads_only_what_is_seen():
    """Pages behind the window may be anyone's, rows past the end anything; a page that is needed and missing is an error."""
    q, kp, vp, table, lens = paged_case(2, [50], 1)
    want = ops.paged_attention(q, kp, vp, table, lens, 10, 3)
    kp2, vp2 = kp.clone(), vp.clone()
    used = {(int(table[0, j // 16]), j % 16) for j in list(range(3)) + list(range(40, 50))}
    for p in range(kp.shape[0]):
        for r in range(16):
            if (p, r) not in used:
                kp2[p, :, r] = float("nan")
                vp2[p, :, r] = float("inf")
    gone = table.clone()
    gone[0, 1] = 99
    assert torch.equal(ops.paged_attention(q, kp2, vp2, gone, lens, 10, 3), want)
    gone[0, 0] = -1
    with pytest.raises(IndexError):
        ops.paged_attention(q, kp, vp, gone, lens, 10, 3)
    assert bool((ops.paged_attention(q, kp, vp, table[:, :0], lens * 0) == 0).all())


@pytest.mark.parametrize("n,window", [(1, None), (3, None), (4, 6)])
def test_infinities_reach_the_tokens_that_see_them(n, window):
    """An infinity or NaN in the newest values and in those that only the oldest token still sees: other tokens are as without it, the
    ones that see it get what the loop's softmax gives."""
    q, kp, vp, table, lens = paged_case(5, [50, 20], n)
    clean = ops.paged_attention(q, kp, vp, table, lens, window)
    for b, L in enumerate(lens.tolist()):
        oldest = 0 if window is None else L - n - window + 1
        for j, d, x in ((L - 1, 0, math.inf), (L - 1, 1, math.nan), (oldest, 2, -math.inf), (L - n, 3, math.inf), (L - n, 4, -math.inf), (oldest, 4, math.inf)):
            vp[table[b, j // 16], :, j % 16, d] = x
    out = ops.paged_attention(q, kp, vp, table, lens, window)
    for b, L in enumerate(lens.tolist()):
        number, row = table[b].long()[torch.arange(L) // 16], torch.arange(L) % 16
        pos, j = L - n + torch.arange(n)[:, None], torch.arange(L)[None]
        seen = j <= pos if window is None else (j <= pos) & (pos - j < window)
        for h in range(4):
            want = loop_attention(q[b, :, h], kp[number, h // 2, row], vp[number, h // 2, row], seen)
            odd = ~torch.isfinite(want)
            assert torch.equal(out[b, :, h].double()[odd].nan_to_num(7.0), want[odd].nan_to_num(7.0)) and int(odd.sum()) >= 4
            assert torch.allclose(out[b, :, h].double()[~odd], want[~odd], rtol=0, atol=64 * U * 8)
    assert n == 1 or torch.equal(out[:, 0, :, 0], clean[:, 0, :, 0])          # the first token does not see the last key


@pytest.mark.parametrize("packed", [False, True])
def test_paged_rope_cache(packed):
    lens, news = [20, 3, 0, 17], [3, 3, 3, 3] if not packed else [4, 3, 0, 1]
    _, kp, vp, table, n = paged_case(3, [20, 3, 1, 17], 1)
    n = torch.tensor(lens, dtype=torch.int32)
    g = torch.Generator().manual_seed(4)
    T = sum(news) + (2 if packed else 0)
    q, k, v = torch.randn(T, 4, 16, generator=g), torch.randn(T, 2, 16, generator=g), torch.randn(T, 2, 16, generator=g)
    cos, sin = ops.precompute_rope_cache(32, 16)
    kw, vw = kp.clone(), vp.clone()
    cu = torch.tensor([0] + news).cumsum(0).to(torch.int32) if packed else None
    out = ops.paged_rope_cache(q, k, v, cos, sin, kp, vp, table, n, cu)
    t, seen = 0, 0
    for b, m in enumerate(news):
        for i in range(m):
            pos = lens[b] - m + i
            if pos < 0:
                assert bool((out[t] == 0).all())
            else:
                turn = lambda x: ops.rope(x[None, None], cos, sin, torch.tensor([[pos]]))[0, 0]  # noqa: E731
                assert torch.equal(out[t], turn(q[t]))
                kw[table[b, pos // 16], :, pos % 16] = turn(k[t])
                vw[table[b, pos // 16], :, pos % 16] = v[t]
                seen += 1
            t += 1
    assert seen and torch.equal(kp, kw) and torch.equal(vp, vw) and bool((out[t:] == 0).all())
    for bad in (lambda: ops.paged_rope_cache(q, k, v, cos, sin, kp, vp, table * 0 - 1, n, cu),
                lambda: ops.paged_rope_cache(q, k, v, cos[:5], sin[:5], kp, vp, table, n, cu)):
        with pytest.raises(IndexError):
            bad()
    if not packed:
        with pytest.raises(RuntimeError):
            ops.paged_rope_cache(q[:11], k[:11], v[:11], cos, sin, kp, vp, table, n)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.paged_rope_cache(q.requires_grad_(), k, v, cos, sin, kp, vp, table, n, cu)


def loop_verify(p, x, u, q=None):
    taken, rows = [], []
    for b in range(p.shape[0]):
        n, V = x.shape[1], p.shape[2]
        r = 0
        while r < n and 0 <= x[b, r] < V and float(u[b, r]) * (float(q[b, r, x[b, r]]) if q is not None else 1.0) < float(p[b, r, x[b, r]]):
            r += 1
        w = [max(float(t), 0.0) if float(t) == float(t) else 0.0 for t in p[b, r]]
        if r < n and 0 <= x[b, r] < V:
            less = [max(float(p[b, r, j]) - float(q[b, r, j]), 0.0) if q is not None else (0.0 if j == x[b, r] else w[j]) for j in range(V)]
            if sum(less) > 0:
                w = less
        total, run, token = sum(w), 0.0, -1
        for j in range(V):
            run += w[j]
            if total > 0 and run > float(u[b, n]) * total:
                token = j
                break
        taken.append(r)
        rows.append([int(t) for t in x[b, :r]] + [token] + [-1] * (n - r))
    return torch.tensor(taken), torch.tensor(rows)


def verify_case(seed, B, n, V, drafts=True, dt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(B, n + 1, V, generator=g)
    p = torch.softmax(base + 0.5 * torch.randn(B, n + 1, V, generator=g), -1).to(dt)
    q = torch.softmax(base[:, :n], -1).to(dt)
    x = torch.multinomial(q.float().reshape(-1, V), 1, generator=g).view(B, n) if drafts and n else q.argmax(-1)
    return p, x, torch.rand(B, n + 1, generator=g), q if drafts else None


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("B,n,V", [(1, 1, 3), (5, 4, 33), (3, 0, 7), (4, 8, 100), (0, 2, 5)])
def test_verify_drafts(B, n, V, drafts):
    p, x, u, q = verify_case(B + n, B, n, V, drafts)
    if n > 1 and B > 1:
        x[1, 1] = -1          # a shorter draft
        x[0, 0] = V           # outside the vocabulary
    got, want = ops.verify_drafts(p, x, u, q), loop_verify(p, x, u, q)
    assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()


def test_verify_drafts_where_nothing_is_left():
    p = torch.tensor([[[0.5, 0.5, 0.0], [0.0, 0.0, 0.0]]])
    assert ops.verify_drafts(p, torch.tensor([[2]]), torch.zeros(1, 2), p[:, :1])[1].tolist() == [[0, -1]]        # residual empty: the target's row
    assert ops.verify_drafts(p, torch.tensor([[0]]), torch.zeros(1, 2))[1].tolist() == [[0, -1]]                 # no weight at all
    assert ops.verify_drafts(p * float("nan"), torch.tensor([[0]]), torch.zeros(1, 2))[1].tolist() == [[-1, -1]]
    with pytest.raises(RuntimeError):
        ops.verify_drafts(p, torch.tensor([[0, 1]]), torch.zeros(1, 2))


def test_random_numbers_outside_their_range():
    """Below zero or NaN: as zero, and never a token without weight.  From one on: the last token with weight."""
    p = torch.tensor([[[0.0, 0.25, 0.5, 0.25, 0.0]]])
    for u, token in ((-1.0, 1), (-math.inf, 1), (math.nan, 1), (0.0, 1), (1 - 2 ** -24, 3), (1.0, 3), (7.0, 3), (math.inf, 3)):
        assert ops.verify_drafts(p, torch.zeros(1, 0, dtype=torch.long), torch.tensor([[u]]))[1].tolist() == [[token]], u


@pytest.mark.parametrize("tokens,uniforms,draft", [(torch.int32, torch.float32, torch.float32), (torch.long, torch.float64, torch.float32),
                                                   (torch.long, torch.float32, torch.bfloat16)])
def test_verify_drafts_refuses_other_types(tokens, uniforms, draft):
    """The same calls as on the device."""
    p, x, u, q = verify_case(1, 2, 3, 11)
    ops.verify_drafts(p, x, u, q)
    with pytest.raises(RuntimeError, match="must be"):
        ops.verify_drafts(p, x.to(tokens), u.to(uniforms), q.to(draft))


def test_verified_drafts_follow_the_target():
    """On a grid of random numbers the outcomes have exactly the target's probabilities (to the grid's step)."""
    p, q = torch.tensor([0.5, 0.25, 0.25]), torch.tensor([0.25, 0.5, 0.25])
    steps = (torch.arange(64) + 0.5) / 64
    u = torch.cartesian_prod(steps, steps)
    count = torch.zeros(3, dtype=torch.float64)
    for x in range(3):
        rows = u.shape[0]
        _, out = ops.verify_drafts(p.expand(rows, 2, 3), torch.full((rows, 1), x), u, q.expand(rows, 1, 3))
        count += float(q[x]) * torch.bincount(out[:, 0], minlength=3).double() / rows
    assert float((count - p.double()).abs().max()) <= 2 / 64


@pytest.mark.parametrize("window,sinks", [(None, 0), (9, 2)])
def test_paged_decoder_follows_the_model(window, sinks):
    """Prompts of different lengths, a sequence that leaves and one that takes its place, drafts right and wrong: the tokens are those of
    the model run over the whole text each time."""
    torch.manual_seed(0)
    model = Llama(llama_tiny_config(vocab_size=61, window=window, attention_sinks=sinks)).eval()
    dec = PagedLlamaDecoder(model, sequences=3, pages=9, page_size=16, max_len=80)
    prompts = [torch.randint(0, 61, (n,), generator=torch.Generator().manual_seed(n)) for n in (5, 33)]
    texts = dict(zip(dec.add(prompts), [p.tolist() for p in prompts]))

    def greedy(text):
        with torch.no_grad():
            return int(model(torch.tensor([text]))[0, -1].argmax())

    def steps(count):
        for _ in range(count):
            went_in = dec.step()
            for b, text in texts.items():
                assert int(went_in[b]) == greedy(text)
                text.append(int(went_in[b]))

    steps(14)
    dec.remove(0)
    del texts[0]
    slot, = dec.add([prompts[0][:2]])
    assert slot == 0
    texts[0] = prompts[0][:2].tolist()
    steps(3)
    # a certain draft (draft_probs None) under u = 0 is taken whatever its probability; under u just below 1 it is refused
    drafts = torch.tensor([[3, 4], [5, 6], [0, 0]])
    uniforms = torch.tensor([[0.0, 1 - 2 ** -24, 0.0], [0.0, 0.0, 0.5], [0.0, 0.0, 0.0]])
    first = dec.tokens[:, 0].tolist()
    taken, out = dec.check(drafts, uniforms, temperature=0.7)
    assert taken.tolist()[:2] == [1, 2] and dec.seq_lens.tolist()[2] == 0
    for b, text in texts.items():
        text += [first[b]] + drafts[b, :int(taken[b])].tolist()
        assert dec.seq_lens[b] == dec.lens[b] == len(text)
        with torch.no_grad():
            p = torch.softmax(model(torch.tensor([text]))[0, -1].double() / 0.7, 0)
        if taken[b] < 2:
            p[drafts[b, taken[b]]] = 0
        run = p.cumsum(0) - float(uniforms[b, 2]) * p.sum()
        assert int(dec.tokens[b]) == int((run > 0).long().argmax())
        text.append(int(dec.tokens[b]))
    went_in = dec.step()
    for b, text in texts.items():
        assert int(went_in[b]) == text[-1] and int(dec.tokens[b]) == greedy(text)
    if window is not None:      # 16-token pages: what lies behind 9 keys and is no sink is back in the pool
        assert all(len(dec._pages[b]) <= 3 for b in texts)
    for b in list(texts):
        dec.remove(b)
    assert sorted(dec.free) == list(range(9)) and all(n is None for n in dec.lens)


def test_paged_decoder_refusals():
    model = Llama(llama_tiny_config(vocab_size=61)).eval()
    dec = PagedLlamaDecoder(model, sequences=1, pages=2, page_size=16, max_len=64)
    with pytest.raises(RuntimeError, match="exhausted"):
        dec.add([torch.zeros(40, dtype=torch.long)])
    with pytest.raises(ValueError, match="max_len"):
        dec.add([torch.zeros(65, dtype=torch.long)])
    with pytest.raises(ValueError, match="at least one"):
        dec.add([torch.zeros(0, dtype=torch.long)])
    assert sorted(dec.free) == [0, 1] and dec.lens == [None]
    dec.add([torch.zeros(31, dtype=torch.long)])
    with pytest.raises(RuntimeError, match="free slots"):
        dec.add([torch.zeros(1, dtype=torch.long)])
    dec.step()
    with pytest.raises(RuntimeError, match="exhausted"):
        dec.step()
    with pytest.raises(ValueError, match="temperature"):
        dec.check(torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, 2), temperature=0.0)
    dec.remove(0)
    with pytest.raises(ValueError, match="not in use"):
        dec.remove(0)


def test_paged_decoder_is_unchanged_by_a_call_that_fails():
    model = Llama(llama_tiny_config(vocab_size=61)).eval()
    dec = PagedLlamaDecoder(model, sequences=2, pages=6, page_size=16, max_len=48)
    with pytest.raises(IndexError):
        dec.add([torch.zeros(3, dtype=torch.long), torch.tensor([61])])      # no such token: the model fails
    assert sorted(dec.free) == list(range(6)) and dec.lens == [None, None] and not dec.active.any()
    dec.add([torch.zeros(3, dtype=torch.long)])
    good = (torch.zeros(2, 2, dtype=torch.long), torch.zeros(2, 3), torch.zeros(2, 2, 61))
    for which, bad in ((0, good[0][:1]), (0, good[0][0]), (1, good[1][:, :2]), (1, good[1].double()), (2, good[2][:, :1]), (2, good[2].bfloat16())):
        args = list(good)
        args[which] = bad
        with pytest.raises(ValueError):
            dec.check(*args)
        assert dec.seq_lens.tolist() == [3, 0] and dec.lens == [3, None]
    taken, _ = dec.check(*good)
    assert dec.lens[0] == 4 + int(taken[0])


class AttnDesc(ctypes.Structure):
    """b200_attn_t of csrc/kernels/b200_kernels.h."""
    _fields_ = ([(n, ctypes.c_int) for n in ("B", "H", "Hkv", "Sq", "Sk", "head_dim", "dtype", "causal")] + [("scale", ctypes.c_float)]
                + [(f"{t}_{d}", ctypes.c_int64) for t in "qkvo" for d in ("sb", "sh", "ss")]
                + [("cu_q", ctypes.c_void_p), ("cu_k", ctypes.c_void_p), ("total_q", ctypes.c_int), ("total_k", ctypes.c_int), ("window", ctypes.c_int),
                   ("sinks", ctypes.c_int), ("workspace", ctypes.c_void_p), ("remainder", ctypes.c_void_p)])


@pytest.mark.parametrize("sinks", [1, 4, 130, 4096, 2 ** 30])
@pytest.mark.parametrize("Hkv", [1, 8, 32])
def test_scratch_of_the_windowed_backward_is_bounded(Hkv, sinks):
    """By the machine, not by sequences times the longest length or by the number of sinks: 1776 pairs of 64 KB."""
    kernels = ctypes.CDLL(os.path.join(os.path.dirname(torch_musa_b200.__file__), "libb200_kernels.so"))
    kernels.b200_flash_attn_bwd_workspace.restype = ctypes.c_int64
    pair = 2 * 128 * 128

    def floats(B, S, window, total=0):
        d = AttnDesc(B=B, H=32, Hkv=Hkv, Sq=S, Sk=S, head_dim=128, dtype=1, causal=1, scale=1.0, total_q=total, total_k=total, window=window, sinks=sinks)
        if total:
            d.cu_q = d.cu_k = 1         # looked at for being there only
        return kernels.b200_flash_attn_bwd_workspace(ctypes.byref(d))

    for window in (1, 64, 128, 1024):
        for B, S, total in ((1, 4096, 0), (1, 32768, 0), (64, 4096, 0), (64, 4096, 4096 + 63 * 100), (200, 8192, 8192 + 199 * 30), (200, 8192, 200 * 8192)):
            n = floats(B, S, window, total)
            assert 0 <= n <= 1776 * pair and n % pair == 0
    assert floats(5, 128, 1) == 0 and floats(3, 100, 1, 300) == 0         # one block of queries is not cut
    if sinks <= 128 and Hkv < 32:
        assert floats(1, 4096, 64) >= 4 * Hkv * pair                        # long ranges of few blocks are


@pytest.mark.parametrize("call,where", [("step", "first layer"), ("step", "head"), ("check", "first layer"), ("check", "head"), ("check", "verification")])
def test_paged_decoder_after_a_step_that_failed_halfway(monkeypatch, call, where):
    """The model or the verification raises when the lengths are already raised: lengths, pages and tokens are as before, and the next call
    goes on as if nothing had been."""
    model = Llama(llama_tiny_config(vocab_size=61)).eval()
    prompts = [torch.arange(15), torch.arange(16), torch.arange(3)]
    dec, other = (PagedLlamaDecoder(model, sequences=4, pages=9, page_size=16, max_len=48) for _ in range(2))
    dec.add(prompts), other.add(prompts)
    args = () if call == "step" else (torch.full((4, 2), 5), torch.full((4, 3), 0.5))
    before = dec.seq_lens.tolist(), list(dec.lens), sorted(dec.free), dec.tokens.tolist(), [dict(p) for p in dec._pages]

    def fails(*_args, **_kw):
        raise RuntimeError("out of memory, say")

    with monkeypatch.context() as m:
        if where == "verification":
            m.setattr("torch_musa_b200.models.paged_decode.BF.verify_drafts", fails)
        else:
            m.setattr(model.layers[0].ffn if where == "first layer" else model.lm_head, "forward", fails)
        with pytest.raises(RuntimeError, match="say"):
            getattr(dec, call)(*args)
    assert (dec.seq_lens.tolist(), list(dec.lens), sorted(dec.free), dec.tokens.tolist(), [dict(p) for p in dec._pages]) == before
    for _ in range(3):
        a, b = getattr(dec, call)(*args), getattr(other, call)(*args)
        for x, y in ((a, b),) if call == "step" else zip(a, b):
            assert torch.equal(x[:3], y[:3])
        assert torch.equal(dec.tokens[:3], other.tokens[:3]) and dec.lens == other.lens == [n or None for n in dec.seq_lens.tolist()]


def test_paged_decoder_refuses_drafts_of_another_type():
    dec = PagedLlamaDecoder(Llama(llama_tiny_config(vocab_size=61)).eval(), sequences=1, pages=4, page_size=16, max_len=48)
    dec.add([torch.arange(4)])
    with pytest.raises(ValueError, match="int64"):
        dec.check(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 3))
    with pytest.raises(ValueError, match="the decoder is on cpu"):
        dec.check(torch.zeros(1, 2, dtype=torch.long), torch.zeros(1, 3, device="meta"))
    assert dec.seq_lens.tolist() == dec.lens == [4] and len(dec.free) == 3


def test_paged_rope_cache_refuses_an_expanded_pool():
    _, kp, vp, table, lens = paged_case(8, [20], 1)
    cos, sin = ops.precompute_rope_cache(32, 16)
    x = torch.randn(1, 4, 16)
    for k, v in ((kp[:, :1].expand_as(kp), vp), (kp, vp[:1].expand_as(vp))):
        with pytest.raises(RuntimeError, match="single memory location"):
            ops.paged_rope_cache(x, x[:, :2], x[:, 2:], cos, sin, k, v, table, lens)
