"""The paged key-value cache on the device: rotary embedding with the cache update, attention of the newest tokens, verification of
drafts, and the decoder that runs them together.

Bounds: with u = eps / 2 of the type, attention keeps its sums and statistics in 32 bits and rounds the output once (the
probabilities are carried to 2^-16): |o - o'| <= u |o| + 2^-13 sum p |v|.  A rotation is two 32-bit products and a sum, rounded
once: u |y| + 2^-22 (|x0 c| + |x1 s|).  Whole numbers are equal."""
import math
import os
import subprocess
import sys

import pytest
import torch

from torch_musa_b200.ops import paged_attention, paged_rope_cache, precompute_rope_cache, verify_drafts

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def case(seed, lens, n, H, Hkv, D, page, dt, window=None, sinks=0, spare=2, order="heads"):
    """q, pools, table, lens on the CPU; every row that no new token sees holds NaN or infinity, and the table entries of pages
    without a visible key are out of range."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-L // page) for L in lens]
    pages, width = sum(need) + spare, max(need) + 1
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), width), 7_000_000, dtype=torch.int32)
    shape = (pages, Hkv, page, D) if order == "heads" else (pages, page, Hkv, D)
    k, v = torch.randn(shape, generator=g).to(dt), torch.randn(shape, generator=g).to(dt)
    if order != "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    seen_rows = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, L in enumerate(lens):
        first = max(0, L - n)
        for j in range(L):
            if window is None or j < sinks or j > first - window:
                p = int(ids[at + j // page])
                table[b, j // page] = p
                seen_rows[p, j % page] = True
        at += need[b]
    hide = (~seen_rows)[:, None, :, None].expand(pages, Hkv, page, D)
    k.masked_fill_(hide, NAN)
    v.masked_fill_(hide, INF)
    q = torch.randn(len(lens), n, H, D, generator=g).to(dt)
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32)


def want_attention(q, k, v, table, lens, window=None, sinks=0, scale=None):
    """(value, bound) in 64 bits."""
    B, n, H, D = q.shape
    Hkv, page = k.shape[1], k.shape[2]
    u = torch.finfo(q.dtype).eps / 2
    out, bound = torch.zeros(B, n, H, D, dtype=torch.float64), torch.zeros(B, n, H, D, dtype=torch.float64)
    for b in range(B):
        L = int(lens[b])
        for i in range(n):
            pos = L - n + i
            at = [j for j in range(pos + 1) if window is None or pos - j < window or j < sinks]
            if not at:
                continue
            number, row = table[b].long()[torch.tensor(at) // page], torch.tensor(at) % page
            kk, vv = k[number, :, row].double().repeat_interleave(H // Hkv, 1), v[number, :, row].double().repeat_interleave(H // Hkv, 1)
            p = torch.softmax(torch.einsum("hd,jhd->hj", q[b, i].double(), kk) * (scale or 1 / math.sqrt(D)), 1)
            out[b, i] = torch.einsum("hj,jhd->hd", p, vv)
            bound[b, i] = u * out[b, i].abs() + 2.0 ** -13 * torch.einsum("hj,jhd->hd", p, vv.abs())
    return out, bound


def check(got, value, bound, what=""):
    over = (got.double().cpu() - value).abs() - bound - 2.0 ** -25
    assert bool((over <= 0).all()), f"{what}: {float(over.nan_to_num(9e9).max())} over the bound"


ATTN = [  # lens, n, H, Hkv, D, page, window, sinks
    ([1], 1, 1, 1, 128, 16, None, 0), ([500], 1, 32, 8, 128, 16, None, 0), ([1, 17, 0, 130], 1, 4, 4, 128, 16, None, 0),
    ([33, 64, 1025], 1, 8, 1, 64, 48, None, 0), ([300, 7, 999], 1, 6, 3, 128, 32, 100, 0), ([300, 7, 999], 1, 6, 2, 64, 32, 100, 4),
    ([40, 200, 5], 5, 4, 1, 128, 16, None, 0), ([40, 200, 3], 5, 8, 2, 64, 64, 17, 3), ([700, 70], 8, 8, 1, 128, 16, 33, 40),
    ([260, 31], 3, 32, 1, 128, 128, 1, 0), ([2500, 1], 1, 4, 2, 128, 16, 2000, 1), ([5000], 2, 2, 2, 128, 64, None, 0), ([90], 40, 4, 2, 64, 16, 20, 1),
    ([2000], 1, 2, 1, 128, 16, 5, 600),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,n,H,Hkv,D,page,window,sinks", ATTN)
def test_paged_attention(bw, dev, dt, lens, n, H, Hkv, D, page, window, sinks):
    args = case(1, lens, n, H, Hkv, D, page, dt, window, sinks)
    out = paged_attention(*(t.to(dev) for t in args), window=window, sinks=sinks)
    bw.synchronize()          # raises if a page that is not needed was asked for
    check(out, *want_attention(*args, window, sinks))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 3])
def test_pages_without_a_visible_key_are_not_asked_for(bw, dev, D, n):
    """Every place of a window's and the sinks' edge within pages of 16, which are shorter than a step of the kernel: the table's other
    entries are out of range, and nothing is reported."""
    for window in (1, 2, 15, 16, 17, 31, 32, 33, 40):
        for sinks in (0, 1, 15, 16, 17, 20):
            lens = [100 + 7 * window % 33, 64, 49, n]
            args = case(window, lens, n, 4, 2, D, 16, torch.float16, window, sinks)
            out = paged_attention(*(t.to(dev) for t in args), window=window, sinks=sinks)
            bw.synchronize()
            check(out, *want_attention(*args, window, sinks), f"window {window}, sinks {sinks}")


def test_other_types_and_head_sizes_take_the_plain_way(bw, dev):
    for dt, D in ((torch.float32, 64), (torch.float16, 32)):
        args = case(20, [40, 3, 0], 2, 4, 2, D, 16, dt, 10, 1)
        out = paged_attention(*(t.to(dev) for t in args), window=10, sinks=1)
        check(out, *want_attention(*args, 10, 1))
    cos, sin = precompute_rope_cache(64, 32)
    _, k, v, table, lens = case(21, [40, 3], 1, 2, 1, 32, 16, torch.float32)
    k.zero_(), v.zero_()
    new = torch.randn(2, 4, 32, generator=torch.Generator().manual_seed(1))
    on = [t.to(dev) for t in (new, cos, sin, k, v, table, lens)]
    out = paged_rope_cache(on[0][:, :2], on[0][:, 2:3], on[0][:, 3:], *on[1:])
    want = paged_rope_cache(new[:, :2], new[:, 2:3], new[:, 3:], cos, sin, k, v, table, lens)
    for a, b in ((out, want), (on[3], k), (on[4], v)):
        assert float((a.cpu() - b).abs().max()) <= 2.0 ** -20      # products of values below 4, each side rounded in 32 bits


def test_infinities_the_plain_way(bw, dev):
    """fp32, several tokens at once: the same pattern of infinities and NaN as off the device."""
    q, k, v, table, lens = case(22, [40, 23], 3, 4, 2, 64, 16, torch.float32, 9, 1)
    hidden = torch.isinf(v)
    for b, L in enumerate(lens.tolist()):
        for j, d, x in ((L - 1, 0, INF), (L - 11, 1, -INF), (L - 3, 2, NAN), (L - 3, 3, INF), (L - 1, 3, -INF)):
            v[table[b, j // 16], :, j % 16, d] = x
    out = paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), window=9, sinks=1).cpu()
    there = table.clamp(0, k.shape[0] - 1)           # off the device an entry that nobody asks for may be anything, too
    want = paged_attention(q, k, v, there, lens, window=9, sinks=1)
    odd = ~torch.isfinite(want)
    assert bool(hidden.any()) and bool(odd.any()) and torch.equal(out[odd].nan_to_num(7.0), want[odd].nan_to_num(7.0))
    assert float((out[~odd] - want[~odd]).abs().max()) <= 2.0 ** -18     # sums of at most 40 products of values below 8, in 32 bits on either side


def test_keys_of_later_tokens_do_not_reach_earlier_ones(bw, dev):
    """n tokens at once with infinities and NaN in the newest keys and values, and in those that only the oldest token still sees."""
    n, window = 4, 50
    q, k, v, table, lens = case(2, [333, 101], n, 8, 2, 128, 16, torch.bfloat16, window, 2)
    clean = paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), window=window, sinks=2).cpu()
    for b, L in enumerate(lens.tolist()):
        for j, x in ((L - 1, NAN), (L - 2, INF), (L - n - window + 1, -INF)):
            v[table[b, j // 16], :, j % 16] = x
            k[table[b, j // 16], :, j % 16] = NAN if j == L - 1 else k[table[b, j // 16], :, j % 16]
    got = paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), window=window, sinks=2).cpu()
    assert torch.equal(got[:, 1], clean[:, 1])
    assert not bool(torch.isfinite(got[:, 0]).any()) and bool(torch.isnan(got[:, 3]).all()) and not bool(torch.isfinite(got[:, 2]).any())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,H,Hkv,D,window", [(1, 4, 2, 128, None), (1, 4, 4, 64, 300), (4, 8, 2, 64, None), (8, 8, 2, 128, 40), (5, 32, 4, 128, None)])
def test_an_infinity_that_a_token_sees_comes_out(bw, dev, dt, n, H, Hkv, D, window):
    """As in the formula: an infinity in a visible value gives an infinity of its sign, both signs or a NaN give NaN, and the other dimensions
    keep their values.  Among the keys that all tokens see, those that some see, and with a probability of 2^-40, which
    fp16 holds as zero."""
    q, k, v, table, lens = case(31, [333, 60], n, H, Hkv, D, 16, dt, window, 2)
    for b, L in enumerate(lens.tolist()):
        for j, d, x in ((L - n - 3, 0, INF), (L - n - 20, 1, -INF), (L - n - 4, 2, INF), (L - n - 19, 2, -INF), (L - 1, 3, INF), (1, 4, -INF), (L - n, 5, NAN)):
            v[table[b, j // 16], :, j % 16, d::16] = x
    faint = int(lens[0]) - n - 9            # its score is -28, the others' are a few
    q[0, :, :, 0], k[..., 0] = 8, 0
    k[table[0, faint // 16], :, faint % 16] = 0
    k[table[0, faint // 16], :, faint % 16, 0] = -3.5 * math.sqrt(D)
    v[table[0, faint // 16], :, faint % 16, 6::16] = INF
    out = paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), window=window, sinks=2).double().cpu()
    bw.synchronize()
    value, bound = want_attention(q, k, v, table, lens, window, 2)
    odd = ~torch.isfinite(value)
    assert bool(odd[..., 6::16][0].all()) and bool(torch.isinf(value[..., 0::16]).all()) and bool(torch.isnan(value[..., 2::16]).all())
    assert torch.equal(torch.isnan(out), torch.isnan(value)) and torch.equal(out[torch.isinf(value)], value[torch.isinf(value)])
    check(out[~odd], value[~odd], bound[~odd])


def test_an_infinity_in_a_very_long_sequence(bw, dev):
    """Where several clusters share the keys and a second kernel joins their parts."""
    q, k, v, table, lens = case(32, [20000], 2, 4, 1, 64, 64, torch.float16)
    for j, d, x in ((3, 0, INF), (19000, 1, -INF), (700, 2, INF), (15000, 2, -INF), (12345, 3, NAN), (19999, 4, INF)):
        v[table[0, j // 64], :, j % 64, d] = x
    out = paged_attention(*(t.to(dev) for t in (q, k, v, table, lens))).cpu().double()
    value, bound = want_attention(q, k, v, table, lens)
    odd = ~torch.isfinite(value)
    assert int(odd.sum()) == 4 * (4 + 5) and torch.equal(out[torch.isinf(value)], value[torch.isinf(value)])
    assert torch.equal(torch.isnan(out), torch.isnan(value))
    check(out[~odd], value[~odd], bound[~odd])


def test_strides_scale_and_slices(bw, dev):
    q, k, v, table, lens = case(3, [130, 47], 2, 4, 2, 128, 32, torch.float16)
    want = paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), softmax_scale=0.2)
    check(want, *want_attention(q, k, v, table, lens, scale=0.2))
    _, k2, v2, _, _ = case(3, [130, 47], 2, 4, 2, 128, 32, torch.float16, order="rows")
    k2.copy_(k), v2.copy_(v)
    rows = [t.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for t in (k2, v2)]            # [pages, page, heads, D] in memory
    wide = torch.full((2, 9), 3, dtype=torch.int32).to(dev)
    wide[:, 2:2 + table.shape[1]] = table.to(dev)
    qq = torch.zeros(2, 2, 8, 128, dtype=torch.float16).to(dev)
    qq[:, :, 4:] = q.to(dev)
    assert torch.equal(paged_attention(qq[:, :, 4:], *rows, wide[:, 2:2 + table.shape[1]], lens.to(dev), softmax_scale=0.2), want)
    odd = torch.zeros(q.numel() + 1, dtype=torch.float16).to(dev)
    odd[1:] = q.to(dev).flatten()
    assert torch.equal(paged_attention(odd[1:].view(q.shape), *rows, table.to(dev), lens.to(dev), softmax_scale=0.2), want)


def test_a_missing_page_is_hidden_and_reported(bw, dev):
    q, k, v, table, lens = case(4, [100, 60], 1, 4, 2, 128, 16, torch.bfloat16)
    bad = table.clone()
    bad[0, 2], bad[1, 3] = -5, k.shape[0]
    out = paged_attention(*(t.to(dev) for t in (q, k, v, bad, lens)))
    with pytest.raises(IndexError):
        bw.synchronize()
    for b, lost in ((0, range(32, 48)), (1, range(48, 60))):       # as a softmax over the other keys
        at = [j for j in range(int(lens[b])) if j not in lost]
        number, row = table[b].long()[torch.tensor(at) // 16], torch.tensor(at) % 16
        kk, vv = (t[number, :, row].double().repeat_interleave(2, 1) for t in (k, v))
        p = torch.softmax(torch.einsum("hd,jhd->hj", q[b, 0].double(), kk) / math.sqrt(128), 1)
        o = torch.einsum("hj,jhd->hd", p, vv)
        check(out[b, 0], o, 2.0 ** -8 * o.abs() + 2.0 ** -13 * torch.einsum("hj,jhd->hd", p, vv.abs()))
    longer = paged_attention(*(t.to(dev) for t in (q, k, v, table[:, :1], lens)))               # a length past the table: its end
    bw.synchronize()
    check(longer, *want_attention(q, k, v, table, lens.clamp_max(16)))


def test_offsets_past_32_bits(bw, dev):
    """A pool of more than 2^31 elements, the pages in use at its end."""
    Hkv, page, D = 8, 64, 128
    pages = 2 ** 31 // (Hkv * page * D) + 40
    q, k, v, table, lens = case(5, [200, 130], 1, 16, Hkv, D, page, torch.bfloat16)
    big = [torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    moved, t = table.clone(), 0
    for b in range(2):
        for i in range(-(-int(lens[b]) // page)):
            moved[b, i] = pages - 1 - 3 * t
            for pool, src in zip(big, (k, v)):
                pool[pages - 1 - 3 * t] = src[table[b, i]].to(dev)
            t += 1
    out = paged_attention(q.to(dev), *big, moved.to(dev), lens.to(dev))
    check(out, *want_attention(q, k, v, table, lens))
    cos, sin = (x.to(dev) for x in precompute_rope_cache(256, D))
    new = torch.randn(2, 3 * Hkv, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(dev)
    paged_rope_cache(new[:, :Hkv], new[:, Hkv:2 * Hkv], new[:, 2 * Hkv:], cos, sin, *big, moved.to(dev), lens.to(dev))
    for b, L in enumerate(lens.tolist()):
        assert torch.equal(big[1][moved[b, (L - 1) // page], :, (L - 1) % page], new[b, 2 * Hkv:])


def test_replay_follows_the_lengths_and_graphs_do_not_share(bw, dev):
    a, b = case(7, [300, 10, 900], 1, 8, 2, 128, 16, torch.bfloat16), case(8, [64, 2000, 5], 1, 8, 2, 128, 16, torch.bfloat16)
    on = [[t.to(dev) for t in x] for x in (a, b)]
    for x in on:
        x[1].nan_to_num_(0.5), x[2].nan_to_num_(0.5, 0.5, 0.5)
    streams, graphs, outs = [bw.Stream(), bw.Stream()], [], []
    for x in on:
        paged_attention(*x)
    bw.synchronize()
    for x in on:
        graph = bw.BlackwellGraph()
        with bw.graph(graph):
            outs.append(paged_attention(*x))
        graphs.append(graph)
    for cut in (0, 3, 63):
        for x, full in zip(on, (a, b)):
            x[4].copy_((full[4] - cut).clamp_min(0))
        bw.synchronize()
        for _ in range(20):
            for s, graph in zip(streams, graphs):
                with bw.stream(s):
                    graph.replay()
        bw.synchronize()
        for x, o in zip(on, outs):
            assert torch.equal(o, paged_attention(*x))


def test_capture_is_the_first_thing_a_program_does(bw, dev):
    """Nothing has run before: torch's CUDA allocator is not set up, and the words that kernels report to are not there."""
    code = """
import torch, torch_musa_b200 as bw
from torch_musa_b200.ops import paged_attention, paged_rope_cache, verify_drafts, window_attention
put = lambda t: t.to("blackwell")
q, pool = put(torch.zeros(1, 1, 2, 64, dtype=torch.float16)), put(torch.ones(4, 2, 16, 64, dtype=torch.float16))
table, lens = put(torch.tensor([[2, 1]], dtype=torch.int32)), put(torch.tensor([20], dtype=torch.int32))
angles, p = put(torch.ones(32, 32)), put(torch.tensor([[[0.0, 1.0]]]))
none, u, x = put(torch.zeros(1, 0, dtype=torch.long)), put(torch.zeros(1, 1)), put(torch.ones(1, 40, 1, 128, dtype=torch.float16))
x.requires_grad_()
graph = bw.BlackwellGraph()
with bw.graph(graph):
    a = paged_rope_cache(q[0], pool[0, :, :1].transpose(0, 1), pool[0, :, :1].transpose(0, 1), angles, angles, pool, pool, table, lens)
    b = paged_attention(q, pool, pool, table, lens)
    c = verify_drafts(p, none, u)[1]
    d = window_attention(x, x, x, 8, 1)
    e = torch.autograd.grad(d, x, d.detach())[0]
graph.replay()
bw.synchronize()
assert bool((a.cpu() == 0).all()) and bool((b.cpu() == 1).all()) and c.tolist() == [[1]] and bool((d.cpu() == 1).all()) and bool(torch.isfinite(e.cpu()).all())
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_very_long_sequences_at_once(bw, dev):
    """Past 16384 keys several clusters share a key head and a second kernel joins their parts: two such calls on two streams, captured
    ones replayed together, lengths that leave most parts without a key."""
    cases = [case(s, [20000], 1, 4, 1, 64, 64, torch.float16) for s in (13, 14)]
    on = [[t.to(dev) for t in c] for c in cases]
    want = [want_attention(*c) for c in cases]
    streams, graphs, outs = [bw.Stream(), bw.Stream()], [], []
    eager = []
    for s, x in zip(streams, on):
        s.wait_stream(bw.current_stream())
        with bw.stream(s):
            eager = eager + [paged_attention(*x)]
    bw.synchronize()
    for e, w in zip(eager, want):
        check(e, *w)
    for x in on:
        graph = bw.BlackwellGraph()
        with bw.graph(graph):
            outs.append(paged_attention(*x))
        graphs.append(graph)
    bw.synchronize()
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with bw.stream(s):
                graph.replay()
    bw.synchronize()
    for o, e in zip(outs, eager):
        assert torch.equal(o, e)
    q, k, v, table, _ = cases[0]
    for n in (0, 1, 70, 700):
        lens = torch.tensor([n], dtype=torch.int32)
        keep = on[0][2].clone().nan_to_num_(0.0, 0.0, 0.0)      # rows past the new end are clean, whatever the case put there
        check(paged_attention(on[0][0], on[0][1], keep, on[0][3], lens.to(dev)), *want_attention(q, k, v, table, lens))


def test_windows_and_sinks_of_any_size(bw, dev):
    q, k, v, table, lens = case(15, [90, 3], 5, 4, 2, 128, 16, torch.bfloat16)
    want = want_attention(q, k, v, table, lens)
    on = [t.to(dev) for t in (q, k, v, table, lens)]
    for window, sinks in ((2 ** 62, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 40)):
        check(paged_attention(*on, window=window, sinks=sinks), *want)


def test_captured_verification(bw, dev):
    p, x, u, q = probs(5, 3, 4, 5000, torch.float32)
    on = [t.to(dev) for t in (p, x, u, q)]
    graph = bw.BlackwellGraph()
    verify_drafts(*on)
    with bw.graph(graph):
        held = verify_drafts(*on)
    for seed in (6, 7):
        new = probs(seed, 3, 4, 5000, torch.float32)
        for a, b in zip(on, new):
            a.copy_(b)
        graph.replay()
        bw.synchronize()
        want = verify_drafts(*new)
        assert torch.equal(held[0].cpu(), want[0]) and torch.equal(held[1].cpu(), want[1])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,news,H,Hkv,D,page,extra", [
    ([1], [1], 1, 1, 128, 16, 0), ([20, 300, 1, 0], [1, 1, 1, 1], 32, 8, 128, 64, 0), ([40, 3, 64], [4, 4, 4], 6, 3, 64, 16, 0),
    ([33, 0, 500, 1], [33, 0, 77, 1], 8, 2, 128, 48, 5), ([200], [150], 2, 1, 64, 32, 1)])
def test_paged_rope_cache(bw, dev, dt, lens, news, H, Hkv, D, page, extra):
    packed = extra > 0
    _, k0, v0, table, n = case(9, [max(x, 1) for x in lens], 1, H, Hkv, D, page, dt)
    k0.zero_(), v0.fill_(3)
    n = torch.tensor(lens, dtype=torch.int32)
    qkv = torch.randn(sum(news) + extra, H + 2 * Hkv, D, generator=torch.Generator().manual_seed(10)).to(dt)
    cos, sin = precompute_rope_cache(512, D)
    cu = torch.tensor([0] + news).cumsum(0).to(torch.int32) if packed else None
    kd, vd = k0.to(dev), v0.to(dev)
    out = paged_rope_cache(*qkv.to(dev).split([H, Hkv, Hkv], 1), cos.to(dev), sin.to(dev), kd, vd, table.to(dev), n.to(dev),
                           cu.to(dev) if packed else None)
    bw.synchronize()
    u = torch.finfo(dt).eps / 2

    def near(got, x, pos):
        c, s, (x0, x1) = cos[pos].double(), sin[pos].double(), x.double().chunk(2, -1)
        for a, b, sign, g in ((x0, x1, -1, got[..., :D // 2]), (x1, x0, 1, got[..., D // 2:])):
            y = a * c + sign * b * s
            check(g, y, u * y.abs() + 2.0 ** -22 * ((a * c).abs() + (b * s).abs()))

    kw, vw, t, out = k0.clone(), v0.clone(), 0, out.cpu()
    for b, m in enumerate(news):
        for i in range(m):
            pos = lens[b] - m + i
            if pos < 0:
                assert bool((out[t] == 0).all())
            else:
                near(out[t], qkv[t, :H], pos)
                where = (table[b, pos // page].long(), slice(None), pos % page)
                near(kd.cpu()[where], qkv[t, H:H + Hkv], pos)
                kw[where], vw[where] = kd.cpu()[where], qkv[t, H + Hkv:]
            t += 1
    assert bool((out[t:] == 0).all()) and torch.equal(vd.cpu(), vw) and torch.equal(kd.cpu(), kw)


def test_paged_rope_cache_reports_what_does_not_fit(bw, dev):
    _, k, v, table, lens = case(11, [40, 20], 1, 2, 1, 128, 16, torch.bfloat16)
    k.zero_(), v.zero_()
    qkv = torch.ones(2, 4, 128, dtype=torch.bfloat16).to(dev)
    cos, sin = (t.to(dev) for t in precompute_rope_cache(64, 128))
    for bad in (-1, k.shape[0]):
        t2 = table.clone()
        t2[0, 2] = bad
        kd, vd = k.to(dev), v.to(dev)
        paged_rope_cache(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], cos, sin, kd, vd, t2.to(dev), lens.to(dev))
        with pytest.raises(IndexError):
            bw.synchronize()
        assert int((vd != 0).any(-1).sum()) == 1        # the other sequence's row
    kd, vd = k.to(dev), v.to(dev)
    paged_rope_cache(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], cos[:30], sin[:30], kd, vd, table.to(dev), lens.to(dev))
    with pytest.raises(IndexError):
        bw.synchronize()
    paged_rope_cache(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], cos, sin, kd, vd, table[:, :2].to(dev), lens.to(dev))
    with pytest.raises(IndexError):
        bw.synchronize()


def probs(seed, B, n, V, dt, drafts=True):
    g = torch.Generator().manual_seed(seed)
    base = 2 * torch.randn(B, n + 1, V, generator=g)
    p = torch.softmax(base + 0.5 * torch.randn(B, n + 1, V, generator=g), -1).to(dt)
    q = torch.softmax(base[:, :n], -1).to(dt)
    x = torch.multinomial(q.float().reshape(-1, V), 1, generator=g).view(B, n) if drafts and n else q.argmax(-1)
    return p, x, torch.rand(B, n + 1, generator=g), q if drafts else None


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,n,V,drafts", [(1, 4, 32000, True), (9, 7, 32000, True), (5, 3, 50257, False), (40, 1, 1000, True), (3, 0, 4001, False),
                                           (7, 8, 5, True), (2, 2, 1, True), (2, 300, 7, True), (130, 2, 129, False)])
def test_verify_drafts(bw, dev, dt, B, n, V, drafts):
    p, x, u, q = probs(B + n + V, B, n, V, dt, drafts)
    if B > 2 and n > 1:
        x[0, 1], x[1, 0], x[2, n - 1] = -1, V, 2 ** 40
    on = [t.to(dev) if t is not None else None for t in (p, x, u, q)]
    got, want = verify_drafts(*on), verify_drafts(p, x, u, q)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("V", [5, 700, 32000])
def test_random_numbers_outside_their_range(bw, dev, V):
    """Each draws a token: what is below zero or NaN counts as zero, from one on it is the last token with weight."""
    us = [-1.0, -INF, NAN, -0.0, 0.0, 1.0, 7.0, INF]
    p = torch.rand(1, 1, V, generator=torch.Generator().manual_seed(V))
    p[..., 0] = p[..., -1] = 0
    args = p.expand(len(us), 1, V).contiguous(), torch.zeros(len(us), 0, dtype=torch.long), torch.tensor(us)[:, None]
    got, want = verify_drafts(*(t.to(dev) for t in args)), verify_drafts(*args)
    assert got[1].flatten().tolist() == want[1].flatten().tolist() == [1] * 5 + [V - 2] * 3 and not got[0].any()


def test_verify_drafts_edges(bw, dev):
    """Random numbers of 0 and just below 1, rows without weight, NaN, views."""
    top = 1 - 2.0 ** -24
    p = torch.tensor([[0.0, 0.25, 0.0, 0.75, 0.0]]).expand(2, 1, 5).contiguous()
    got = verify_drafts(p.to(dev), torch.zeros(2, 0, dtype=torch.long).to(dev), torch.tensor([[0.0], [top]]).to(dev))
    assert got[1].tolist() == [[1], [3]] and got[0].tolist() == [0, 0]
    p = torch.tensor([[[0.5, 0.5, 0.0], [0.0, 0.0, 0.0]]])
    zero, on = torch.zeros(1, 2), p.to(dev)
    assert verify_drafts(on, torch.tensor([[2]]).to(dev), zero.to(dev), on[:, :1])[1].tolist() == [[0, -1]]
    assert verify_drafts(on, torch.tensor([[0]]).to(dev), zero.to(dev))[1].tolist() == [[0, -1]]
    assert verify_drafts(on * NAN, torch.tensor([[0]]).to(dev), zero.to(dev))[1].tolist() == [[-1, -1]]
    p, x, u, q = probs(3, 6, 4, 700, torch.float32)
    wide = torch.zeros(6, 9, 900).to(dev)
    wide[:, 3:8, 100:800] = p.to(dev)
    want = verify_drafts(p, x, u, q)
    got = verify_drafts(wide[:, 3:8, 100:800], x.to(dev).t().contiguous().t(), u.to(dev).t().contiguous().t(), q.to(dev))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_refusals(bw, dev):
    q, k, v, table, lens = (t.to(dev) for t in case(12, [40], 1, 4, 2, 128, 16, torch.bfloat16))
    cos, sin = (t.to(dev) for t in precompute_rope_cache(64, 128))
    new = q[:, 0]
    for bad in (lambda: paged_attention(q[:, :, :3], k, v, table, lens), lambda: paged_attention(q, k[:, :, :8], v[:, :, :8], table, lens),
                lambda: paged_attention(q, k, v.half(), table, lens), lambda: paged_attention(q, k, v, table.long(), lens),
                lambda: paged_attention(q, k, v, table, lens.cpu()), lambda: paged_attention(q, k, v, table[0], lens),
                lambda: paged_attention(q, k, v, table, lens.repeat(2)), lambda: paged_attention(q[0], k, v, table, lens),
                lambda: paged_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, table, lens),
                lambda: paged_attention(q.clone().requires_grad_(), k, v, table, lens),
                lambda: paged_rope_cache(new, new, new, cos, sin, k, v, table, lens),
                lambda: paged_rope_cache(new, new[:, :2], new[:, :2], cos.half(), sin.half(), k, v, table, lens),
                lambda: paged_rope_cache(new, new[:, :2], new[:, :2], cos[:, :32], sin[:, :32], k, v, table, lens),
                lambda: paged_rope_cache(new, new[:, :2], new[:, :2], cos, sin, k, v, table, lens, lens),
                lambda: verify_drafts(torch.ones(1, 3, 5).to(dev), torch.zeros(1, 2).to(dev), torch.zeros(1, 3).to(dev)),
                lambda: verify_drafts(torch.ones(1, 3, 5).to(dev), torch.zeros(1, 2, dtype=torch.long).to(dev), torch.zeros(1, 2).to(dev)),
                lambda: verify_drafts(torch.ones(1, 3, 5).to(dev), torch.zeros(1, 2, dtype=torch.long), torch.zeros(1, 3).to(dev)),
                lambda: verify_drafts(torch.ones(1, 3, 5).to(dev), torch.zeros(1, 2, dtype=torch.long).to(dev), torch.zeros(1, 3).to(dev),
                                      torch.ones(1, 2, 4).to(dev))):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        paged_attention(q, k, v, table, lens, window=0)
    assert paged_attention(q[:0], k, v, table[:0], lens[:0]).shape == (0, 1, 4, 128)
    assert paged_attention(q[:, :0], k, v, table, lens).shape == (1, 0, 4, 128)


@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 3)])
def test_decoder_captured_step_and_checked_drafts(bw, dev, window, sinks):
    """The captured step gives the eager step's tokens; drafts that are the model's own greedy tokens, checked at a low temperature,
    are taken, and the cache then continues as if they had been decoded one by one."""
    from torch_musa_b200.models import Llama, LlamaConfig, PagedLlamaDecoder

    cfg = LlamaConfig(vocab_size=256, dim=512, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=512, max_seq_len=400, window=window, attention_sinks=sinks)
    torch.manual_seed(0)
    model = Llama(cfg).to(torch.bfloat16).eval().to(dev)
    model.reset_parameters(std=0.2)
    prompts = [torch.randint(0, 256, (n,), generator=torch.Generator().manual_seed(n)) for n in (150, 1, 40)]

    def decoder(graph):
        d = PagedLlamaDecoder(model, sequences=4, pages=40, page_size=16, device=dev)
        if graph:
            d.capture()
        assert d.add(prompts) == [0, 1, 2]
        return d

    a, b = decoder(False), decoder(True)
    eager = torch.stack([a.step() for _ in range(60)], 1)[:3].cpu()
    replayed = torch.stack([b.step() for _ in range(60)], 1)[:3].cpu()
    assert torch.equal(eager, replayed)
    c = decoder(False)
    first = torch.stack([c.step() for _ in range(20)], 1)[:3].cpu()
    assert torch.equal(first, eager[:, :20])
    drafts = torch.zeros(4, 5, dtype=torch.long)
    drafts[:3] = eager[:, 21:26]
    drafts[1, 3] = -1                                    # a shorter draft
    taken, out = c.check(drafts.to(dev), torch.full((4, 6), 0.5).to(dev), temperature=1e-3)
    for s, t in enumerate(taken.tolist()[:3]):
        # what was taken was the greedy text (a near tie may stop a draft early; it cannot take a wrong token)
        assert t <= (3 if s == 1 else 5) and out[s, :t].tolist() == eager[s, 21:21 + t].tolist()
        assert c.seq_lens[s] == c.lens[s] == prompts[s].numel() + 21 + t
    assert sum(taken.tolist()[:3]) >= 6
    full = [s for s in range(3) if out[s, taken[s]] == eager[s, 21 + int(taken[s])]]
    went_in = c.step()
    assert all(int(went_in[s]) == int(out[s, taken[s]]) for s in range(3)) and full
    bw.synchronize()


def test_decoder_is_unchanged_by_drafts_that_are_refused(bw, dev):
    from torch_musa_b200.models import Llama, LlamaConfig, PagedLlamaDecoder

    cfg = LlamaConfig(vocab_size=64, dim=256, n_layers=1, n_heads=4, n_kv_heads=2, ffn_dim=256, max_seq_len=64)
    torch.manual_seed(0)
    d = PagedLlamaDecoder(Llama(cfg).to(torch.bfloat16).eval().to(dev), sequences=2, pages=6, page_size=16, device=dev)
    d.add([torch.arange(15)])
    drafts, uniforms = torch.zeros(2, 2, dtype=torch.long, device=dev), torch.zeros(2, 3, device=dev)
    for bad in ((drafts.int(), uniforms), (drafts.cpu(), uniforms), (drafts, uniforms.cpu()), (drafts, uniforms, torch.zeros(2, 2, 64))):
        with pytest.raises(ValueError):
            d.check(*bad)
        assert d.seq_lens.tolist() == [15, 0] and d.lens == [15, None] and len(d.free) == 5
    taken, _ = d.check(drafts, uniforms)
    assert d.seq_lens.tolist() == [16 + int(taken[0]), 0] and d.lens == [16 + int(taken[0]), None]


def test_an_expanded_pool_is_read_but_not_written(bw, dev):
    q, k, v, table, lens = (t.to(dev) for t in case(33, [40], 1, 4, 2, 64, 16, torch.bfloat16))
    cos, sin = (t.to(dev) for t in precompute_rope_cache(64, 64))
    new, one = q[:, 0], k[:, :1]
    assert torch.equal(paged_attention(q, one.expand_as(k), v, table, lens), paged_attention(q, one.repeat(1, 2, 1, 1), v, table, lens))
    for pools in ((one.expand_as(k), v), (k, v[:1].expand_as(v))):
        with pytest.raises(RuntimeError, match="single memory location"):
            paged_rope_cache(new, new[:, :2], new[:, 2:], cos, sin, *pools, table, lens)
