"""Causal attention with a sliding window and sinks on the tensor-core kernels, dense and packed, against the formulas in 64 bits.

Tolerances are bounds, not guesses.  With u = eps / 2 of the type, the kernels round P (and in the backward P and dS) to the type
before a product and every result once; sums are 32-bit.  So |o - o'| <= u (sum p |v| + |o|), |dV - dV'| <= u (sum p |dO| + |dV|),
and dS carries u |dS| and scale p e with e = sum_d (error of o_d) |dO_d|, the error of the row sums that the backward forms from
the rounded o.  Beside them stands 2^-14 of the same sums for the 32-bit parts, and 2^-25 for each value below fp16's normal range (its steps there are 2^-24): per term of a sum, and once for the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


def visible(sq, sk, window, sinks):
    i, j = torch.arange(sq)[:, None], torch.arange(sk)[None, :]
    m = j <= i
    return m if window is None else m & ((i - j < window) | (j < sinks))


def formula(q, k, v, do, window, sinks, scale=None):
    """One sequence: q [Sq, H, D], k / v [Sk, Hkv, D] in any type.  Returns {name: (value, bound)} in 64 bits."""
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25
    c = u + 2.0 ** -14
    H, Hkv = q.shape[1], k.shape[1]
    G, scale = H // Hkv, scale if scale is not None else 1 / math.sqrt(D)
    seen = visible(q.shape[0], k.shape[0], window, sinks)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    r = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    for h in range(H):
        qh, kh, vh, gh = q[:, h], k[:, h // G], v[:, h // G], do[:, h]
        s = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
        top = s.amax(1, keepdim=True) if s.shape[1] else s.new_zeros(s.shape[0], 1)
        p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
        p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
        o = p @ vh
        e_o = c * (p @ vh.abs() + o.abs()) + tiny * (seen.double() @ vh.abs())
        ds = p * (gh @ vh.T - (gh * o).sum(1, keepdim=True)) * scale
        e_ds = c * ds.abs() + scale * p * (e_o * gh.abs()).sum(1, keepdim=True) + 2.0 ** -14 * scale * p * (gh.abs() @ vh.abs().T) + tiny * seen.double()
        dq, dk, dv = ds @ kh, ds.T @ qh, p.T @ gh
        for n, at, val, err in (("o", h, o, e_o), ("dq", h, dq, e_ds @ kh.abs() + u * dq.abs()), ("dk", h // G, dk, e_ds.T @ qh.abs()),
                                ("dv", h // G, dv, c * (p.T @ gh.abs()) + tiny * (seen.double().T @ gh.abs()))):
            r[n][0][:, at] += val
            r[n][1][:, at] += err
    for n in ("dk", "dv"):
        r[n][1] += u * r[n][0].abs()
    return r


def check(got, want, what):
    value, bound = want
    over = (got.double().cpu() - value).abs() - bound - 2.0 ** -25
    assert bool((over <= 0).all()), f"{what}: {float(over.max())} over the bound, at {tuple(int(x) for x in torch.nonzero(over == over.max())[0])}"


def inputs(dt, q_shape, k_shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda s: torch.randn(*s, generator=g).to(dt)  # noqa: E731
    return mk(q_shape), mk(k_shape), mk(k_shape), mk(q_shape)


DENSE = [  # B, Sq, Sk, H, Hkv, window, sinks
    (1, 1, 1, 1, 1, 1, 0), (1, 5, 5, 2, 1, 1, 0), (2, 128, 128, 2, 2, 128, 0), (1, 129, 129, 2, 1, 128, 1), (1, 300, 300, 4, 2, 1, 4),
    (2, 511, 511, 2, 2, 64, 0), (1, 640, 640, 4, 1, 130, 130), (1, 777, 777, 2, 1, 257, 3), (1, 1024, 1024, 2, 2, 256, 300),
    (1, 1400, 1400, 2, 1, 100, 5), (1, 400, 400, 2, 2, 100000, 7), (1, 700, 200, 2, 1, 64, 0), (1, 700, 200, 2, 1, 64, 2), (1, 130, 600, 2, 2, 50, 129),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Sq,Sk,H,Hkv,window,sinks", DENSE)
def test_dense_forward_and_gradients(bw, dev, dt, B, Sq, Sk, H, Hkv, window, sinks):
    from torch_musa_b200.ops import window_attention

    q, k, v, do = inputs(dt, (B, Sq, H, D), (B, Sk, Hkv, D))
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    before = bw._C._native_sdp_forward_calls(), bw._C._native_sdp_backward_calls()
    out = window_attention(*leaves, window, sinks)
    grads = torch.autograd.grad(out, leaves, do.to(dev))
    assert (bw._C._native_sdp_forward_calls(), bw._C._native_sdp_backward_calls()) == (before[0] + 1, before[1] + 1)
    bw.synchronize()
    assert bw._C._gemm_status(False) == 0
    for b in range(B):
        want = formula(q[b], k[b], v[b], do[b], window, sinks)
        for n, got in zip(("o", "dq", "dk", "dv"), (out, *grads)):
            check(got.detach()[b], want[n], n)


PACKED = [  # lengths of the queries, lengths of the keys, H, Hkv, window, sinks, rows past the last sequence
    ([1], None, 2, 1, 3, 0, 0), ([300, 1, 129, 64], None, 4, 2, 100, 3, 0), ([200, 333], None, 2, 2, 257, 130, 70), ([0, 260, 0, 5], None, 2, 1, 32, 1, 3),
    ([900, 17], None, 2, 1, 64, 4, 200), ([400, 100], [90, 500], 2, 1, 40, 0, 1), ([64, 30], [0, 30], 2, 1, 40, 2, 0),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,klens,H,Hkv,window,sinks,extra", PACKED)
def test_packed_sequences(bw, dev, dt, lens, klens, H, Hkv, window, sinks, extra):
    """Rows past the last sequence hold NaN: they reach nobody, and get zeros."""
    from torch_musa_b200.ops import flash_attn_varlen_func

    klens = klens or lens
    q, k, v, do = inputs(dt, (sum(lens) + extra, H, D), (sum(klens) + extra, Hkv, D))
    for t, n in ((q, lens), (k, klens), (v, klens), (do, lens)):
        t[sum(n):] = float("nan")
    cq = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    ck = torch.tensor([0] + klens).cumsum(0).to(torch.int32)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    out = flash_attn_varlen_func(*leaves, cq.to(dev), ck.to(dev), max(lens), max(klens), causal=True, window=window, sinks=sinks)
    grads = torch.autograd.grad(out, leaves, do.to(dev))
    bw.synchronize()
    assert bw._C._gemm_status(False) == 0
    got = [t.detach().cpu() for t in (out, *grads)]
    for i in range(len(lens)):
        a, b = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        want = formula(q[a], k[b], v[b], do[a], window, sinks)
        for n, t, rows in zip(("o", "dq", "dk", "dv"), got, (a, a, b, b)):
            check(t[rows], want[n], f"sequence {i}, {n}")
    for t, n in zip(got, (lens, lens, klens, klens)):
        assert bool((t[sum(n):] == 0).all())


@pytest.mark.parametrize("sinks", [0, 5])
@pytest.mark.parametrize("empty", ["front", "back", "spread"])
def test_many_packed_sequences(bw, dev, empty, sinks):
    """More sequences than a warp has lanes, dozens of them empty: where the units of work are counted."""
    g = torch.Generator().manual_seed(1)
    some = torch.randint(1, 40, (40,), generator=g).tolist() + [300]
    lens = {"front": [0] * 70 + some, "back": some + [0] * 70, "spread": [n for x in some for n in (0, x, 0)]}[empty]
    test_packed_sequences(bw, dev, torch.float16, lens, None, 2, 1, 30, sinks, 9)


@pytest.mark.parametrize("bad", [0, 1])
@pytest.mark.parametrize("packed", [False, True])
def test_infinities_and_nan_stay_in_their_sequence(bw, dev, packed, bad):
    """One of two sequences holds infinities and NaN near its ends; nothing of the other changes.  (dq is a sum of at most three blocks in
    any order: its 32-bit values differ by 2^-22 of the sum of their sizes, which is below 2^-18 of the largest value here, and by a step
    of the type when that moves a rounding.)"""
    from torch_musa_b200.ops import flash_attn_varlen_func, window_attention

    S, H, Hkv, dt = 200, 2, 1, torch.bfloat16
    clean = inputs(dt, (2, S, H, D), (2, S, Hkv, D), 31)
    dirty = [t.clone() for t in clean]
    for t in dirty:
        t[bad, S - 1], t[bad, S - 3], t[bad, 0] = math.inf, math.nan, -math.inf
    cu = torch.tensor([0, S, 2 * S], dtype=torch.int32).to(dev)

    def run(tensors):
        q, k, v, do = (t.flatten(0, 1).to(dev) if packed else t.to(dev) for t in tensors)
        for t in (q, k, v):
            t.requires_grad_()
        o = flash_attn_varlen_func(q, k, v, cu, cu, S, S, causal=True, window=50, sinks=3) if packed else window_attention(q, k, v, 50, 3)
        return [t.detach().cpu().view(2, S, -1, D)[1 - bad].float() for t in (o, *torch.autograd.grad(o, (q, k, v), do))]

    want, got = run(clean), run(dirty)
    for name, a, b in zip(("o", "dq", "dk", "dv"), want, got):
        if name == "dq":
            assert bool(((a - b).abs() <= 2.0 ** -7 * a.abs() + 2.0 ** -18 * a.abs().max()).all())
        else:
            assert torch.equal(a, b), name


def test_a_window_longer_than_the_sequence_is_the_causal_mask(bw, dev):
    """Bit for bit: the same blocks in the same order."""
    import torch.nn.functional as F
    from torch_musa_b200.ops import flash_attn_varlen_func, window_attention

    q, k, v, _ = (t.to(dev) for t in inputs(torch.bfloat16, (2, 515, 4, D), (2, 515, 2, D)))
    want = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True, enable_gqa=True).transpose(1, 2)
    assert torch.equal(window_attention(q, k, v, 515), want)
    cu = torch.tensor([0, 515, 1030], dtype=torch.int32).to(dev)
    flat = [t.reshape(1030, -1, D) for t in (q, k, v)]
    assert torch.equal(flash_attn_varlen_func(*flat, cu, cu, 515, 515, causal=True, window=600).view_as(want), want)
    assert torch.equal(flash_attn_varlen_func(*flat, cu, cu, 515, 515, causal=True).view_as(want), want)


def test_strided_broadcast_and_odd_operands(bw, dev):
    """Views of one fused projection, an expanded head, and rows that do not start on 16 bytes."""
    from torch_musa_b200.ops import window_attention

    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(2, 260, 8, D, generator=g).to(torch.bfloat16)
    q, k, v = qkv.split([4, 2, 2], 2)
    plain = window_attention(*(t.contiguous().to(dev) for t in (q, k, v)), 70, 2)
    dq, dk, dv = qkv.to(dev).split([4, 2, 2], 2)
    assert torch.equal(window_attention(dq, dk, dv, 70, 2), plain)
    one = k[:, :, :1].contiguous().to(dev)
    assert torch.equal(window_attention(dq, one.expand(-1, -1, 2, -1), dv, 70, 2), window_attention(dq, one.repeat(1, 1, 2, 1), dv, 70, 2))
    odd = torch.zeros(q.numel() + 1, dtype=torch.bfloat16)
    odd[1:] = q.flatten()
    assert torch.equal(window_attention(odd.to(dev)[1:].view(q.shape), dk, dv, 70, 2), plain)
    leaf = one.clone().requires_grad_()          # the gradient of a broadcast head is the sum over its copies
    grad = torch.autograd.grad(window_attention(dq, leaf.expand(-1, -1, 2, -1), dv, 70, 2), leaf, torch.ones_like(plain))[0]
    assert grad.shape == one.shape


def test_gradients_against_differences(bw, dev):
    """Along a random direction, the change of a weighted output over a step of 2^-4 (exact in bf16 for inputs that are
    multiples of 2^-3): the formula's curvature and the rounding of the outputs bound what differs."""
    from torch_musa_b200.ops import window_attention

    g = torch.Generator().manual_seed(5)
    S, window, sinks, h = 200, 60, 2, 2.0 ** -4
    x = [(torch.randint(-8, 9, (1, S, n, D), generator=g) / 8.0) for n in (2, 1, 1)]
    w = torch.randn(1, S, 2, D, generator=g).to(torch.bfloat16)
    leaves = [t.to(torch.bfloat16).to(dev).requires_grad_() for t in x]
    grads = torch.autograd.grad(window_attention(*leaves, window, sinks), leaves, w.to(dev))
    bound = formula(*(t[0].to(torch.bfloat16) for t in x), w[0], window, sinks)
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randint(0, 2, x[i].shape, generator=g) * 2.0 - 1
        ends = []
        for sign in (1, -1):
            moved = [t.clone() for t in x]
            moved[i] = moved[i] + sign * h * d
            ends.append([t[0].double() for t in moved])
        f = [float((formula(*e, w[0].double(), window, sinks)["o"][0] * w[0].double()).sum()) for e in ends]
        third = [float((formula(*[t[0].double() + s * 2 * h * d[0].double() * (j == i) for j, t in enumerate(x)], w[0].double(), window, sinks)["o"][0] * w[0].double()).sum()) for s in (1, -1)]
        slope = (f[0] - f[1]) / (2 * h)
        coarse = (third[0] - third[1]) / (4 * h)
        got = float((grads[i].double().cpu()[0] * d[0].double()).sum())
        # the error of a central difference is a quarter of the step-2h one's, so it is at most the distance of the two
        allowed = abs(slope - coarse) + float((bound[n][1] * d[0].abs().double()).sum())
        assert abs(got - slope) <= allowed, (n, got, slope, allowed)


def test_captured_forward_and_backward_replay(bw, dev):
    from torch_musa_b200.ops import window_attention

    q, k, v, do = (t.to(dev) for t in inputs(torch.bfloat16, (1, 300, 2, D), (1, 300, 1, D)))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    step = lambda: (lambda o: [o.detach(), *torch.autograd.grad(o, leaves, do)])(window_attention(*leaves, 64, 3))  # noqa: E731
    side = bw.Stream()
    side.wait_stream(bw.current_stream())
    with bw.stream(side):
        step()
    bw.current_stream().wait_stream(side)
    graph = bw.BlackwellGraph()
    with bw.graph(graph):
        held = step()
    for seed in (1, 2):
        new = [t.to(dev) for t in inputs(torch.bfloat16, (1, 300, 2, D), (1, 300, 1, D), seed)]
        with torch.no_grad():
            for leaf, t in zip(leaves, new):
                leaf.copy_(t)
        do.copy_(new[3])
        graph.replay()
        bw.synchronize()
        got = [t.clone() for t in held]
        want = step()
        for n, (a, b) in enumerate(zip(got, want)):
            if n == 1:       # dq: 32-bit sums in the order of arrival, rounded once
                assert float((a.double() - b.double()).abs().max()) <= float(2 ** -8 * b.double().abs().max())
            else:
                assert torch.equal(a, b)


def test_llama_with_a_window_trains_like_the_plain_model(bw, dev):
    """The model's attention goes through the operator; logits follow the same model on the CPU in 32 bits."""
    from torch_musa_b200.models import Llama, LlamaConfig

    cfg = LlamaConfig(vocab_size=64, dim=256, n_layers=2, n_heads=2, n_kv_heads=1, ffn_dim=256, max_seq_len=256, window=40, attention_sinks=2)
    torch.manual_seed(0)
    model = Llama(cfg).to(torch.bfloat16)
    tokens = torch.randint(0, 64, (2, 200), generator=torch.Generator().manual_seed(1))
    cpu = Llama(cfg)
    cpu.load_state_dict(model.state_dict())
    want = cpu(tokens)
    before = bw._C._native_sdp_forward_calls()
    loss = model.to(dev)(tokens.to(dev), tokens.to(dev))
    loss.backward()
    assert bw._C._native_sdp_forward_calls() == before + cfg.n_layers
    got = model(tokens.to(dev)).float().cpu()
    # 16 roundings of 2^-8 along the way (norms, projections, residuals of two layers), each at most the values' own size
    assert float((got - want).abs().max()) <= 16 * 2 ** -8 * float(want.abs().max())
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in model.parameters())


def test_backward_is_refused_where_determinism_is_asked_for(bw, dev):
    from torch_musa_b200.ops import flash_attn_varlen_func, window_attention

    q, k, v, do = (t.to(dev) for t in inputs(torch.bfloat16, (1, 40, 2, D), (1, 40, 1, D)))
    q.requires_grad_()
    cu = torch.tensor([0, 40], dtype=torch.int32).to(dev)
    outs = [window_attention(q, k, v, 8), flash_attn_varlen_func(q[0], k[0], v[0], cu, cu, 40, 40, causal=True, window=8)]
    torch.use_deterministic_algorithms(True)
    try:
        for out in outs:
            with pytest.raises(RuntimeError, match="deterministic"):
                out.sum().backward()
    finally:
        torch.use_deterministic_algorithms(False)


def test_refusals(bw, dev):
    from torch_musa_b200.ops import window_attention

    op = torch.ops.blackwell
    q, k, v, do = (t.to(dev) for t in inputs(torch.bfloat16, (1, 40, 4, D), (1, 40, 2, D)))
    out, lse = op.window_attention(q, k, v, 8)
    for bad in (lambda: op.window_attention(q, k, v, 0), lambda: op.window_attention(q, k, v, 8, -1), lambda: op.window_attention(q, k, v, 8, 0, 0.0),
                lambda: op.window_attention(q, k, v[:, :30], 8), lambda: op.window_attention(q, k.half(), v, 8), lambda: op.window_attention(q, k.cpu(), v, 8),
                lambda: op.window_attention(q[:, :, :3], k, v, 8), lambda: op.window_attention(q[..., :64], k[..., :64], v[..., :64], 8),
                lambda: op.window_attention_backward(do[:, :20], q, k, v, out, lse, 8), lambda: op.window_attention_backward(do, q, k, v, out, lse.half(), 8),
                lambda: op.varlen_attention(q[0], k[0], v[0], *[torch.tensor([0, 40], dtype=torch.int32).to(dev)] * 2, 40, 40, False, None, 8)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        window_attention(q, k, v, 8, softmax_scale=-1.0)
    leaf = q.clone().requires_grad_()
    grad = torch.autograd.grad(window_attention(leaf, k, v, 8).sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):           # no second order
        grad.sum().backward()
    for shape_q, shape_k in (((1, 0, 4, D), (1, 5, 2, D)), ((0, 5, 4, D), (0, 5, 2, D)), ((2, 5, 4, D), (2, 0, 2, D))):
        e = [torch.zeros(s, dtype=torch.float16).to(dev).requires_grad_() for s in (shape_q, shape_k, shape_k)]
        o = window_attention(*e, 3)
        assert o.shape == shape_q and bool((o == 0).all())
        assert [g.shape for g in torch.autograd.grad(o, e, torch.zeros_like(o))] == [t.shape for t in e]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_remainder_of_the_output(bw, dev, dt):
    """Equal scores: every probability is one before the division, so only the output itself is rounded, and output + remainder is off by
    the rounding of the remainder (u of it, u^2 of the output, 2^-25 below fp16's normal range) and by four 32-bit roundings."""
    S, H, Hkv = 200, 4, 2
    _, k, v, do = inputs(dt, (1, S, H, D), (1, S, Hkv, D), 6)
    q = torch.zeros(1, S, H, D, dtype=dt)
    p = visible(S, S, 3, 1).double()
    vv = v[0].double().repeat_interleave(H // Hkv, 1)
    want = torch.einsum("ij,jhd->ihd", p / p.sum(1, keepdim=True), vv)
    bound = (torch.finfo(dt).eps / 2) ** 2 * want.abs() + 2.0 ** -22 * torch.einsum("ij,jhd->ihd", p, vv.abs()) + 2.0 ** -25
    op, on = torch.ops.blackwell, [t.to(dev) for t in (q, k, v, do)]
    out, lse, rest = op.window_attention_with_remainder(*on[:3], 3, 1)
    assert bool(((out.cpu().double() + rest.cpu().double())[0] - want).abs().le(bound).all()) and bool(rest.any())
    plain = op.window_attention(*on[:3], 3, 1)
    assert torch.equal(plain[0], out) and torch.equal(plain[1], lse)
    cu = torch.tensor([0, S], dtype=torch.int32).to(dev)
    more = [torch.cat((t[0], torch.full_like(t[0, :7], float("nan")))) for t in on[:3]]
    o2, l2, r2 = op.varlen_attention_with_remainder(*more, cu, cu, S, S, 3, 1)
    assert torch.equal(o2[:S], out[0]) and torch.equal(r2[:S], rest[0]) and not o2[S:].any() and not r2[S:].any()
    grads = op.window_attention_backward(on[3], *on[:3], out, lse, 3, 1, None, rest)
    apart = op.window_attention_backward(on[3], *on[:3], out, lse, 3, 1, None, rest.transpose(1, 2).contiguous().transpose(1, 2))
    for a, b in zip(grads[1:], apart[1:]):      # another layout of the remainder; dq depends on the order of arrival
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="remainder"):
        op.window_attention_backward(on[3], *on[:3], out, lse, 3, 1, None, rest[:, :100])
    for empty in ((0, S), (1, 0)):
        e = torch.empty(*empty, H, D, dtype=dt, device=dev)
        assert op.window_attention_with_remainder(e, e, e, 3, 1)[2].shape == e.shape


@pytest.mark.parametrize("lens,window,sinks", [([1], 7, 0), ([1, 1, 1], 300, 4), ([300], 1, 0), ([129, 1, 40], 1, 0)])
def test_a_query_with_one_key_has_no_gradient_through_its_score(bw, dev, lens, window, sinks):
    """The softmax over one key is constant, so the gradients of q and k are zero, exactly."""
    from torch_musa_b200.ops import flash_attn_varlen_func

    q, k, v, do = (t.to(dev) for t in inputs(torch.bfloat16, (sum(lens), 4, D), (sum(lens), 2, D), 5))
    for t in (q, k, v):
        t.requires_grad_()
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    o = flash_attn_varlen_func(q, k, v, cu, cu, max(lens), max(lens), causal=True, window=window, sinks=sinks)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    assert not dq.any() and not dk.any() and torch.equal(o, v.repeat_interleave(2, 1))
    assert torch.allclose(dv.float(), do.float().view(-1, 2, 2, D).sum(2), rtol=2.0 ** -8, atol=2.0 ** -8)


def test_other_types_and_head_sizes_take_the_plain_way(bw, dev):
    from torch_musa_b200.ops import flash_attn_varlen_func, window_attention

    g = torch.Generator().manual_seed(9)
    for dt, size in ((torch.float32, 128), (torch.bfloat16, 64)):
        q, k, v, do = (torch.randn(1, 50, h, size, generator=g).to(dt) for h in (4, 2, 2, 4))
        sides = []
        for where in (dev, torch.device("cpu")):
            leaves = [t.to(where).requires_grad_() for t in (q, k, v)]
            out = window_attention(*leaves, 9, 2)
            flat = [t[0].to(where) for t in (q, k, v)]
            cu = torch.tensor([0, 20, 50], dtype=torch.int32).to(where)
            packed = flash_attn_varlen_func(*flat, cu, cu, 30, 30, causal=True, window=9, sinks=2)
            sides.append([t.detach().cpu().float() for t in (out, packed, *torch.autograd.grad(out, leaves, do.to(where)))])
        for a, b in zip(*sides):      # both ways round to the type a few times, values of a few
            assert float((a - b).abs().max()) <= 16 * torch.finfo(dt).eps * max(1.0, float(b.abs().max()))


def test_two_streams_and_two_graphs(bw, dev):
    """Forward and backward of two problems at once, each on a stream of its own, eager and replayed: scratch is not shared.  (The last
    bits of dq follow the order of arrival.)"""
    from torch_musa_b200.ops import window_attention

    cases = [inputs(torch.bfloat16, (1, 700, 4, D), (1, 700, 2, D), s) for s in (1, 2)]
    cases = [[t.to(dev) for t in c] for c in cases]
    leaves = [[t.clone().requires_grad_() for t in c[:3]] for c in cases]
    step = lambda i: (lambda o: [o.detach(), *torch.autograd.grad(o, leaves[i], cases[i][3])])(window_attention(*leaves[i], 100, 5))  # noqa: E731
    want = [step(i) for i in range(2)]
    streams = [bw.Stream(), bw.Stream()]
    bw.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with bw.stream(s):
                got[i] = step(i)
    graphs, held = [], []
    for i in range(2):
        graph = bw.BlackwellGraph()
        with bw.graph(graph):
            held.append(step(i))
        graphs.append(graph)
    bw.synchronize()
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with bw.stream(s):
                graph.replay()
    bw.synchronize()
    for i in range(2):
        for result in (got[i], held[i]):
            for n, (a, b) in enumerate(zip(result, want[i])):
                if n == 1:
                    assert float((a.double() - b.double()).abs().max()) <= float(2 ** -8 * b.double().abs().max())
                else:
                    assert torch.equal(a, b)


@pytest.mark.parametrize("sinks", [0, 3])
def test_small_gradients_of_a_long_window(bw, dev, sinks):
    """fp16, thousands of keys and an incoming gradient of 2^-10: what is rounded before the products, p (dP - delta) without the softmax
    scale, still has most of its bits.  The formula in 64 bits with that one rounding, and that of the result, gives the error to
    expect (as a norm); the sums of 32 bits and the output's remainder stay far below it, so twice it is the limit.  (With the scale in
    front of the rounding it is eleven times as large.)"""
    from torch_musa_b200.ops import window_attention

    S, H, window, dt, scale = 2600, 2, 2500, torch.float16, 1 / math.sqrt(D)
    q, k, v, do = inputs(dt, (1, S, H, D), (1, S, 1, D), 41)
    do = (do.float() * 2.0 ** -10).to(dt)
    seen = visible(S, S, window, sinks)
    want, model = [torch.zeros(S, n, D, dtype=torch.float64) for n in (H, 1)], [torch.zeros(S, n, D, dtype=torch.float64) for n in (H, 1)]
    for h in range(H):
        qh, kh, vh, gh = q[0, :, h].double(), k[0, :, 0].double(), v[0, :, 0].double(), do[0, :, h].double()
        p = torch.softmax((qh @ kh.T * scale).masked_fill(~seen, -math.inf), 1)
        ds = p * (gh @ vh.T - (gh * (p @ vh)).sum(1, keepdim=True))
        for to, x in ((want, ds), (model, ds.to(dt).double())):
            to[0][:, h] = x @ kh * scale
            to[1][:, 0] += x.T @ qh * scale
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*leaves, window, sinks), leaves, do.to(dev))
    for name, got, w, m in zip(("dq", "dk"), grads, want, model):
        expected = float((m.to(dt).double() - w).norm())
        assert float((got[0].cpu().double() - w).norm()) <= 2 * expected, name


@pytest.mark.parametrize("lens,H,Hkv,window,sinks", [
    ([1500] + [40, 7, 129] * 12, 2, 1, 64, 4), ([40, 0, 129] * 12 + [1500], 2, 2, 64, 4), ([60, 1400, 3, 0, 900, 128], 4, 2, 100, 130),
    ([300, 1300, 1], 2, 1, 64, 1000), ([260, 1300], 2, 2, 1, 5000), ([1100] * 3, 16, 16, 40, 1100)])
def test_chunks_of_the_sinks_go_by_the_sequence(bw, dev, lens, H, Hkv, window, sinks):
    """Long sequences among short ones, sinks over many blocks and past every end: each sequence's own number of chunks, in places that
    follow from its first row."""
    test_packed_sequences(bw, dev, torch.bfloat16, lens, None, H, Hkv, window, sinks, 3)


@pytest.mark.parametrize("B,S,H,Hkv,window,sinks", [(2, 1000, 2, 1, 64, 1000), (1, 1400, 16, 16, 64, 4000), (1, 1100, 2, 2, 1, 300)])
def test_many_sinks(bw, dev, B, S, H, Hkv, window, sinks):
    test_dense_forward_and_gradients(bw, dev, torch.float16, B, S, S, H, Hkv, window, sinks)


def test_scratch_does_not_grow_with_the_number_of_sequences(bw, dev):
    """One long sequence among 199 short ones: what the backward allocates beside its results follows the rows."""
    from torch_musa_b200.ops import flash_attn_varlen_func

    lens, H, Hkv = [8192] + [20] * 199, 8, 8
    n = sum(lens)
    q, k, v, do = (torch.ones(n, h, D, dtype=torch.bfloat16, device=dev) for h in (H, Hkv, Hkv, H))
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    for t in (q, k, v):
        t.requires_grad_()
    out = flash_attn_varlen_func(q, k, v, cu, cu, 8192, 8192, causal=True, window=128, sinks=4)
    bw.synchronize()
    bw.reset_peak_memory_stats()
    before = bw.memory_allocated()
    torch.autograd.grad(out, (q, k, v), do)
    bw.synchronize()
    results = 2 * D * n * (H + 2 * Hkv) + 4 * D * n * H + 4 * n * H          # gradients, dq and the row dots in 32 bits
    assert bw.max_memory_allocated() - before <= results + 1776 * 2 * 4 * 128 * 128


@pytest.mark.parametrize("sinks", [0, 2])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
def test_reach_of_what_is_not_finite_within_a_sequence(bw, dev, which, sinks):
    """A NaN at place 300, block 2 of a sequence of eight blocks, window 4.  Queries of blocks 2 and 3 see keys of block 2, and queries of
    block 2 see keys of blocks 1 and 2 (and the sinks' block 0): nothing else changes.  (dq is a sum of at most three blocks in any order,
    as in the test of two sequences above.)"""
    from torch_musa_b200.ops import window_attention

    S, H, at, dt = 1000, 2, 300, torch.bfloat16
    clean = dict(zip(("q", "k", "v", "do"), inputs(dt, (1, S, H, D), (1, S, H, D), 51)))
    dirty = {n: t.clone() for n, t in clean.items()}
    dirty[which][0, at] = math.nan

    def run(x):
        leaves = [x[n].to(dev).requires_grad_() for n in ("q", "k", "v")]
        o = window_attention(*leaves, 4, sinks)
        return dict(zip(("o", "dq", "dk", "dv"), (t.detach().cpu()[0].float() for t in (o, *torch.autograd.grad(o, leaves, x["do"].to(dev))))))

    want, got = run(clean), run(dirty)
    place = torch.arange(S) // 128
    by_key = {"o": (place == 2) | (place == 3), "dq": (place == 2) | (place == 3), "dk": place == 2, "dv": place == 2}
    by_query = {"o": place == 2, "dq": place == 2, "dk": (place == 1) | (place == 2) | ((place == 0) & (sinks > 0)),
                "dv": (place == 1) | (place == 2) | ((place == 0) & (sinks > 0))}
    for n in want:
        rows = (by_key if which in ("k", "v") else by_query)[n].clone()
        if n in ("dk", "dv") and which in ("k", "v"):      # a query that has become NaN reaches the keys of its own blocks
            rows |= by_query[n] | (place == 3)
        a, b = want[n][~rows], got[n][~rows]
        if n == "dq":
            assert bool(((a - b).abs() <= 2.0 ** -7 * a.abs() + 2.0 ** -18 * a.abs().max()).all())
        else:
            assert torch.equal(a, b), n
    seen = {"q": ("o", at), "k": ("o", at), "v": ("o", at + 3), "do": ("dv", at - 3)}[which]
    assert bool(got[seen[0]][seen[1]].isnan().all())


def test_second_order_of_packed_sequences_is_refused(bw, dev):
    """As of a dense batch, instead of a gradient with a part missing; the first order with a graph is as without."""
    from torch_musa_b200.ops import flash_attn_varlen_func

    q, k, v, do = (t.to(dev) for t in inputs(torch.bfloat16, (40, 2, D), (40, 1, D)))
    for t in (q, k, v):
        t.requires_grad_()
    cu = torch.tensor([0, 15, 40], dtype=torch.int32).to(dev)
    out = flash_attn_varlen_func(q, k, v, cu, cu, 25, 25, causal=True, window=8, sinks=1)
    plain = torch.autograd.grad(out, (k, v), do, retain_graph=True)
    grads = torch.autograd.grad(out, (k, v), do, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    with pytest.raises(RuntimeError):           # no graph behind them: the incoming gradient is a constant
        grads[0].float().sum().backward()
    out = flash_attn_varlen_func(q, k, v, cu, cu, 25, 25, causal=True, window=8, sinks=1)
    grads = torch.autograd.grad(out.float().square().sum(), (k, v), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grads[0].float().sum().backward()
