"""Windowed attention with sinks, forward and backward, against the formula in 64 bits.

Bounds by element. Half a step of bf16 is 2^-8 of the value (HALF). The probabilities go into their products in bf16, so a result is off by at most HALF times the
sum of its terms' sizes, and by HALF of itself when it is rounded. dS = P (dP - delta) takes over what delta is off by: delta is the sum of dO O with the O that
the forward pass rounded. What is summed and exponentiated in fp32 adds at most SLACK = 2^-14 of the terms' sizes: the scores' own error, up to 128 products of
a few units rounded to 2^-24, times the scale, is below 2^-15 in an exponent. As a norm over many independent roundings the same errors are smaller
by a factor of at least sqrt(3) each; three of them in a row stay below HALF."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF, SLACK, HD = 2.0 ** -8, 2.0 ** -14, 128


def _heads(qkv, B, S, nh, nkv):
    x = qkv.double().view(B, S, nh + 2 * nkv, HD).transpose(1, 2)
    rep = nh // nkv
    return x[:, :nh], x[:, nh:nh + nkv].repeat_interleave(rep, 1), x[:, nh + nkv:].repeat_interleave(rep, 1)


def _mask(S, window, sinks, device="cuda"):
    i, j = torch.arange(S, device=device)[:, None], torch.arange(S, device=device)[None]
    return (j <= i) & ((j > i - window) | (j < sinks))


def _forward(qkv, B, S, nh, nkv, window, sinks, scale):
    q, k, v = _heads(qkv, B, S, nh, nkv)
    s = (q @ k.transpose(2, 3) * scale).masked_fill(~_mask(S, window, sinks), -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    return p, p @ v, lse


def _flat(x):
    B, h, S, d = x.shape
    return x.transpose(1, 2).reshape(B * S, h * d)


def _grouped(x, nkv):
    B, nh, S, d = x.shape
    return x.view(B, nkv, nh // nkv, S, d).sum(2)


def _reference(qkv, dout, B, S, nh, nkv, window, sinks, scale):
    """out, lse, dqkv and how far each element of out and dqkv may be off."""
    q, k, v = _heads(qkv, B, S, nh, nkv)
    p, o, lse = _forward(qkv, B, S, nh, nkv, window, sinks, scale)
    o_tol = (HALF + SLACK) * (p @ v.abs()) + HALF * o.abs()
    do = dout.double().view(B, S, nh, HD).transpose(1, 2)
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    # of one dS: its rounding, what delta is off by, what dP and P are
    ds_tol = HALF * ds.abs() + p * (do.abs() * o_tol).sum(-1, keepdim=True) + SLACK * p * (do.abs() @ v.abs().transpose(2, 3))
    dq, dk, dv = scale * ds @ k, _grouped(scale * ds.transpose(2, 3) @ q, nkv), _grouped(p.transpose(2, 3) @ do, nkv)
    dq_tol = scale * ds_tol @ k.abs() + (HALF + SLACK) * dq.abs()
    dk_tol = _grouped(scale * ds_tol.transpose(2, 3) @ q.abs(), nkv) + (HALF + SLACK) * dk.abs()
    dv_tol = _grouped((HALF + SLACK) * p.transpose(2, 3) @ do.abs(), nkv) + HALF * dv.abs()
    return _flat(o), _flat(o_tol), lse, _flat(torch.cat([dq, dk, dv], 1)), _flat(torch.cat([dq_tol, dk_tol, dv_tol], 1))


def _inputs(B, S, nh, nkv, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(B * S, (nh + 2 * nkv) * HD, device="cuda", generator=g) * size).to(torch.bfloat16)
    return qkv, torch.randn(B * S, nh * HD, device="cuda", generator=g).to(torch.bfloat16)


SHAPES = [(1, 1, 1, 1, 1, 0), (3, 1, 4, 2, 5, 3), (2, 5, 2, 1, 2, 1), (1, 127, 3, 1, 128, 0), (2, 128, 2, 2, 1, 0), (1, 129, 4, 1, 64, 4), (2, 200, 8, 1, 37, 130),
          (1, 300, 2, 1, 300, 300), (1, 513, 6, 2, 128, 1), (2, 640, 4, 4, 129, 127), (1, 1000, 9, 3, 200, 0), (1, 1300, 4, 1, 16, 129), (1, 1111, 16, 2, 4096, 5),
          (5, 256, 3, 3, 255, 256), (30, 384, 3, 1, 100, 2), (1, 2049, 4, 2, 640, 64), (1, 3000, 2, 1, 50, 1), (65535, 2, 2, 1, 2, 1), (1, 150, 128, 1, 40, 2),
          (1, 128, 32, 8, 128, 1), (1, 333, 8, 1, 512, 1)]


@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", SHAPES)
def test_forward_and_backward(B, S, nh, nkv, window, sinks):
    from cai_b200 import ops
    qkv, dout = _inputs(B, S, nh, nkv)
    scale = HD ** -0.5
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks)
    o, o_tol, l, d, d_tol = _reference(qkv, dout, B, S, nh, nkv, window, sinks, scale)
    assert ((out.double() - o).abs() <= o_tol).all()
    assert ((lse.double() - l).abs() <= 2.0 ** -15 * (1 + l.abs())).all()
    assert ((dqkv.double() - d).abs() <= d_tol).all()
    if S >= 100:
        assert (out.double() - o).norm() <= HALF * o.norm()
        cols = torch.tensor([0, nh, nh + nkv, nh + 2 * nkv]) * HD
        for a, b in zip(cols[:-1], cols[1:]):
            if window > 1 or a == nh * HD + nkv * HD:     # of a window of one nothing is left of dq and dk but its rounding
                assert (dqkv[:, a:b].double() - d[:, a:b]).norm() <= HALF * d[:, a:b].norm()
    assert torch.equal(dqkv, ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks)), "the same bits in every run"


@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", [(1, 1500, 2, 1, 200, 3), (1, 6000, 3, 1, 128, 130), (2, 900, 4, 2, 900, 0), (1, 9000, 2, 2, 1000, 40),
                                                     (1, 4100, 8, 1, 1, 1), (1, 2500, 1, 1, 385, 257)])
def test_exactly_the_visible_keys_count(B, S, nh, nkv, window, sinks):
    """With q = k = 0 every visible key weighs 1 / n. V and dO say which class (row mod 128) a row is of: n times the output has to be the whole
    number of visible keys of each class, and dV the sum of 1 / n over the queries of a class. At most 128 rows of a class count, half a step of
    bf16 of that is half a row; sums above that are compared within it."""
    from cai_b200 import ops
    eye = torch.eye(HD, device="cuda").repeat((S + HD - 1) // HD, 1)[:S]
    qkv = torch.zeros(B, S, nh + 2 * nkv, HD, device="cuda", dtype=torch.bfloat16)
    qkv[:, :, nh + nkv:] = eye[:, None]
    qkv = qkv.view(B * S, -1)
    dout = eye[:, None].expand(B, S, nh, HD).reshape(B * S, -1).to(torch.bfloat16).contiguous()
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks)
    seen = _mask(S, window, sinks).double()
    n = seen.sum(1)
    assert torch.allclose(lse.double(), n.log().expand(B, nh, S), rtol=2.0 ** -20, atol=2.0 ** -20)
    counts = seen @ eye.double()
    got = out.double().view(B, S, nh, HD) * n[:, None, None]
    assert ((got - counts[:, None]).abs() <= HALF * counts[:, None]).all() and counts.max() * HALF < 0.5
    dv = (seen / n[:, None]).t() @ eye.double() * (nh // nkv)
    # a probability of 1 / n is rounded to bf16, and so is the sum
    assert ((dqkv.view(B, S, -1, HD)[:, :, nh + nkv:].double() - dv[:, None]).abs() <= (2 * HALF + SLACK) * dv[:, None]).all()


@pytest.mark.parametrize("S,nh,nkv,window,sinks", [(700, 2, 1, 100, 3), (1500, 3, 3, 300, 130)])
def test_visible_keys_in_dq(S, nh, nkv, window, sinks):
    """Uniform weights again (q = 0): K says which class a key is of, and one column of V whether it is odd; dq is then the number of visible odd keys of a class less its
    share, over n."""
    from cai_b200 import ops
    eye = torch.eye(HD, device="cuda").repeat((S + HD - 1) // HD, 1)[:S]
    odd = (torch.arange(S, device="cuda") // HD % 2).float()
    qkv = torch.zeros(S, nh + 2 * nkv, HD, device="cuda")
    qkv[:, nh:nh + nkv] = eye[:, None]
    qkv[:, nh + nkv:, 0] = odd[:, None]
    qkv = qkv.view(S, -1).to(torch.bfloat16)
    dout = torch.zeros(S, nh, HD, device="cuda", dtype=torch.bfloat16)
    dout[..., 0] = 1.0
    dout = dout.view(S, -1)
    out, lse = ops.flash_attn_window_fwd(qkv, 1, S, nh, nkv, HD, window, sinks, scale=1.0)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, 1, S, nh, nkv, HD, window, sinks, scale=1.0)
    seen = _mask(S, window, sinks).double()
    p = seen / seen.sum(1, keepdim=True)
    mean = p @ odd.double()
    terms = p * (odd.double() - mean[:, None])
    tol = (3 * HALF) * (p @ eye.double())       # dS, the rounded mean in it, dq: terms are at most p
    assert ((dqkv.view(S, -1, HD)[:, :nh].double() - (terms @ eye.double())[:, None]).abs() <= tol[:, None]).all()


def test_it_is_causal_attention_where_the_window_covers_the_sequence():
    from cai_b200 import ops
    B, S, nh, nkv = 2, 512, 4, 2
    qkv, dout = _inputs(B, S, nh, nkv, 3)
    out, lse = ops.flash_attn_fwd(qkv, B, S, nh, nkv, HD)
    o, _, _, d, d_tol = _reference(qkv, dout, B, S, nh, nkv, S, 0, HD ** -0.5)
    for window, sinks in ((S, 0), (10 * S, 7), (2 ** 31 - 1, 2 ** 31 - 1), (1, S)):
        out_w, lse_w = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
        assert (out_w.double() - out.double()).norm() <= HALF * out.double().norm()
        assert torch.allclose(lse_w, lse, rtol=2.0 ** -15, atol=2.0 ** -15)
        dqkv = ops.flash_attn_window_bwd(qkv, out_w, dout, lse_w, B, S, nh, nkv, HD, window, sinks)
        assert ((dqkv.double() - d).abs() <= d_tol).all()


def test_large_and_far_apart_scores():
    """Rows with one dominant key, scores of many hundreds, hidden keys larger than all visible ones."""
    from cai_b200 import ops
    B, S, nh, nkv, window, sinks = 1, 500, 2, 1, 70, 2
    qkv, dout = _inputs(B, S, nh, nkv, 5)
    x = qkv.view(S, nh + 2 * nkv, HD)
    x[:, :nh] *= 8
    x[::50, nh] *= 30          # keys whose scores reach hundreds wherever they are seen, and more where they are hidden
    scale = HD ** -0.5
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks)
    p, o, l = _forward(qkv, B, S, nh, nkv, window, sinks, scale)
    v = _heads(qkv, B, S, nh, nkv)[2]
    # a score is a sum of 128 products in fp32, then scaled in another rounding or two: off by 2^-22 of its terms' sizes at most on average, 2^-20 allowed
    q, k, _ = _heads(qkv, B, S, nh, nkv)
    s_off = 2.0 ** -20 * (q.abs() @ k.abs().transpose(2, 3) * scale).masked_fill(~_mask(S, window, sinks), 0).amax(-1, keepdim=True)
    tol = (HALF + SLACK + 2 * s_off) * (p @ v.abs()) + HALF * o.abs()
    assert ((out.double() - _flat(o)).abs() <= _flat(tol)).all()
    assert ((lse.double() - l).abs() <= s_off[..., 0] + 2.0 ** -20 * l.abs()).all()
    assert torch.isfinite(dqkv).all()
    d = _reference(qkv, dout, B, S, nh, nkv, window, sinks, scale)[3]
    assert (dqkv.double() - d).norm() <= 2 * HALF * d.norm()


def test_the_gradient_against_differences():
    """A central difference of the formula in 64 bits along a direction, against the gradient's product with it, within what its elements may be off."""
    from cai_b200 import ops
    B, S, nh, nkv, window, sinks = 2, 150, 4, 2, 33, 5
    qkv, dout = _inputs(B, S, nh, nkv, 7)
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks).double()
    d_tol = _reference(qkv, dout, B, S, nh, nkv, window, sinks, HD ** -0.5)[4]

    def loss(x):
        return (_flat(_forward(x, B, S, nh, nkv, window, sinks, HD ** -0.5)[1]) * dout.double()).sum()
    for seed in range(3):
        u = torch.randn(qkv.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed), dtype=torch.float64)
        h = 1e-5
        slope = (loss(qkv.double() + h * u) - loss(qkv.double() - h * u)) / (2 * h)
        # the errors of many elements, along a random direction, add up like their norm: four times that
        assert (slope - (dqkv * u).sum()).abs() <= 4 * d_tol.norm() + 1e-6 * slope.abs()


def test_pitches_and_neighbours():
    """Rows inside a larger buffer whose other columns and rows hold NaN, and the gradient's rows inside another: nothing else is read or written."""
    from cai_b200 import ops
    B, S, nh, nkv, window, sinks = 3, 77, 2, 1, 20, 2
    cols = (nh + 2 * nkv) * HD
    qkv, dout = _inputs(B, S, nh, nkv, 9)
    big = torch.full((B * S + 200, cols + 24), float("nan"), device="cuda", dtype=torch.bfloat16)
    big[:B * S, 8:8 + cols] = qkv
    view = big[:B * S, 8:8 + cols]
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    out_v, lse_v = ops.flash_attn_window_fwd(view, B, S, nh, nkv, HD, window, sinks)
    assert torch.equal(out, out_v) and torch.equal(lse, lse_v)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks)
    d_big = torch.full((B * S + 130, cols + 40), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.flash_attn_window_bwd(view, out, dout, lse, B, S, nh, nkv, HD, window, sinks, dqkv=d_big[:B * S, 16:16 + cols])
    assert torch.equal(d_big[:B * S, 16:16 + cols], dqkv)
    d_big[:B * S, 16:16 + cols] = 7.0
    assert (d_big == 7.0).all()
    # a sequence that is not finite leaves the others as they are
    bad = qkv.clone()
    bad[S:2 * S] = float("nan")
    out_b, lse_b = ops.flash_attn_window_fwd(bad, B, S, nh, nkv, HD, window, sinks)
    keep = torch.arange(B * S, device="cuda") // S != 1
    assert torch.equal(out_b[keep], out[keep]) and torch.equal(lse_b[[0, 2]], lse[[0, 2]])
    d_bad = ops.flash_attn_window_bwd(bad, out_b, dout, lse_b, B, S, nh, nkv, HD, window, sinks)
    assert torch.equal(d_bad[keep], dqkv[keep])


def test_workspaces_given_and_streams_side_by_side():
    """Two calls at once on two streams, each with workspaces of its own, the same as one after the other; the scratch may hold anything."""
    from cai_b200 import ops
    B, S, nh, nkv, window, sinks = 1, 3000, 8, 1, 200, 130
    a = [_inputs(B, S, nh, nkv, seed) for seed in (1, 2)]
    fwd = [ops.flash_attn_window_fwd(q, B, S, nh, nkv, HD, window, sinks) for q, _ in a]
    want = [ops.flash_attn_window_bwd(q, o, d, l, B, S, nh, nkv, HD, window, sinks) for (q, d), (o, l) in zip(a, fwd)]
    need = ops.flash_attn_window_bwd_scratch(B, S, nh, nkv, window, sinks)
    assert need > 0
    work = [(torch.full((B, nh, S), float("nan"), device="cuda"), torch.full((need // 4,), float("nan"), device="cuda")) for _ in a]
    got = [torch.full_like(w, float("nan")) for w in want]
    streams = [torch.cuda.Stream() for _ in a]
    torch.cuda.synchronize()
    for _ in range(3):
        for (q, d), (o, l), (delta, scratch), g, st in zip(a, fwd, work, got, streams):
            with torch.cuda.stream(st):
                ops.flash_attn_window_bwd(q, o, d, l, B, S, nh, nkv, HD, window, sinks, dqkv=g, delta=delta, scratch=scratch)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert torch.equal(w, g)
    with pytest.raises(ops.KernelError, match="scratch"):
        ops.flash_attn_window_bwd(a[0][0], *fwd[0][:1], a[0][1], fwd[0][1], B, S, nh, nkv, HD, window, sinks, scratch=work[0][1][1:])


@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", [(3, 700, 4, 2, 1, 1), (2, 1001, 3, 3, 2, 0), (1, 3000, 8, 1, 3, 4), (40, 900, 6, 2, 8, 16), (9, 17, 4, 4, 17, 0), (5, 96, 4, 1, 50, 9),
                                                     (64, 33, 8, 8, 33, 33), (1, 2000, 2, 1, 20, 4), (2, 97, 8, 2, 97, 0)])
def test_few_visible_keys_are_no_less_exact(B, S, nh, nkv, window, sinks):
    """dS is a difference of two numbers that are alike where few keys are visible: row sums that have the rounding of out in them would leave dq and dk two to three
    roundings off. They are off by two independent ones, their operand's and their own: as norms sqrt(2) of one; 1.6 for values that lie unevenly between powers of two."""
    from cai_b200 import ops
    qkv, dout = _inputs(B, S, nh, nkv, 21)
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks).double()
    d = _reference(qkv, dout, B, S, nh, nkv, window, sinks, HD ** -0.5)[3]
    cols = [0, nh * HD, (nh + nkv) * HD, (nh + 2 * nkv) * HD]
    for a, b in zip(cols, cols[1:]):
        once = (d[:, a:b].to(torch.bfloat16).double() - d[:, a:b]).norm()
        assert (dqkv[:, a:b] - d[:, a:b]).norm() <= 1.6 * once


@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", [(1, 900, 2, 1, 900, 0), (1, 4000, 1, 1, 4000, 0), (2, 1500, 8, 1, 100, 100), (1, 333, 8, 1, 512, 1), (1, 6000, 2, 2, 1000, 17),
                                                     (1, 129, 32, 8, 129, 1), (1, 5000, 4, 2, 300, 257)])
def test_what_the_scratch_held_does_not_matter(B, S, nh, nkv, window, sinks):
    """Sums cut over heads, over query tiles, over both, and the sinks' rows alone: what is joined is what the parts wrote."""
    from cai_b200 import ops
    qkv, dout = _inputs(B, S, nh, nkv, 5)
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    need = ops.flash_attn_window_bwd_scratch(B, S, nh, nkv, window, sinks)
    assert need > 0
    got = [ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks, scratch=torch.full((need // 4,), v, device="cuda"),
                                     dqkv=torch.full_like(qkv, v)) for v in (float("nan"), 0.0)]
    assert got[0].isfinite().all() and torch.equal(*got)


def test_offsets_beyond_32_bits():
    """More than 2^31 elements in one sequence: its end gives what the end alone gives, bit for bit (the cut lies at a tile's beginning)."""
    from cai_b200 import ops
    S, nh, nkv, window, tail = 384 * 1024, 32, 8, 200, 2048
    cols = (nh + 2 * nkv) * HD
    assert S * cols > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(3)
    piece = torch.randn(4096, cols, device="cuda", generator=g).to(torch.bfloat16)
    qkv = piece.repeat(S // 4096, 1)
    dout = torch.randn(4096, nh * HD, device="cuda", generator=g).to(torch.bfloat16).repeat(S // 4096, 1)
    out, lse = ops.flash_attn_window_fwd(qkv, 1, S, nh, nkv, HD, window)
    q, d = qkv[S - tail:].contiguous(), dout[S - tail:].contiguous()
    o, l = ops.flash_attn_window_fwd(q, 1, tail, nh, nkv, HD, window)
    assert torch.equal(out[S - tail + window:], o[window:]) and torch.equal(lse[..., S - tail + window:], l[..., window:])
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, 1, S, nh, nkv, HD, window)
    dq = ops.flash_attn_window_bwd(q, o, d, l, 1, tail, nh, nkv, HD, window)
    # (sums may be cut otherwise in the short call: their order is that of fp32 additions, their result is rounded once)
    a, b = dqkv[S - tail + window:].float(), dq[window:].float()
    assert ((a - b).abs() <= 2 * HALF * b.abs() + SLACK * b.abs().amax()).all()


def test_captured_and_replayed():
    from cai_b200 import ops
    B, S, nh, nkv, window, sinks = 2, 700, 4, 1, 130, 3
    qkv, dout = _inputs(B, S, nh, nkv, 11)

    def step():
        out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
        return out, lse, ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (12, 13):
        q, d = _inputs(B, S, nh, nkv, seed)
        qkv.copy_(q)
        dout.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, step()):
            assert torch.equal(x, y)


def test_gradients_over_what_is_read_are_refused():
    """dqkv in qkv's, out's or dout's place; beside qkv in one buffer it is taken."""
    from cai_b200 import ops
    S, nh, nkv, cols = 150, 2, 1, 4 * HD
    both = torch.randn(S, 2 * cols, device="cuda").to(torch.bfloat16)
    qkv, dqkv = both[:, :cols], both[:, cols:]
    dout = torch.randn(S, nh * HD, device="cuda").to(torch.bfloat16)
    out, lse = ops.flash_attn_window_fwd(qkv, 1, S, nh, nkv, HD, 20)
    want = ops.flash_attn_window_bwd(qkv, out, dout, lse, 1, S, nh, nkv, HD, 20)
    for bad in (qkv, both[:, HD:HD + cols], both[:, cols - 8:2 * cols - 8]):
        with pytest.raises(ops.KernelError, match="shares memory"):
            ops.flash_attn_window_bwd(qkv, out, dout, lse, 1, S, nh, nkv, HD, 20, dqkv=bad)
    wide = torch.empty(S * cols, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError, match="shares memory"):
        ops.flash_attn_window_bwd(qkv, out, wide[:S * nh * HD].view(S, nh * HD), lse, 1, S, nh, nkv, HD, 20, dqkv=wide.view(S, cols))
    assert ops.flash_attn_window_bwd(qkv, out, dout, lse, 1, S, nh, nkv, HD, 20, dqkv=dqkv) is dqkv
    assert torch.equal(dqkv, want)


def test_no_rows():
    from cai_b200 import ops
    for B, S in ((0, 5), (3, 0)):
        qkv = torch.zeros(0, 4 * HD, device="cuda", dtype=torch.bfloat16)
        out, lse = ops.flash_attn_window_fwd(qkv, B, S, 2, 1, HD, 4, 1)
        assert out.shape == (0, 2 * HD) and lse.shape == (B, 2, S)
        assert ops.flash_attn_window_bwd(qkv, out, out, lse, B, S, 2, 1, HD, 4, 1).shape == qkv.shape


def test_tensors_elsewhere_are_refused():
    from cai_b200 import ops
    qkv, dout = _inputs(1, 8, 2, 1)
    out, lse = ops.flash_attn_window_fwd(qkv, 1, 8, 2, 1, HD, 4)
    with pytest.raises(ops.KernelError, match="current device"):
        ops.flash_attn_window_fwd(qkv.cpu(), 1, 8, 2, 1, HD, 4)
    with pytest.raises(ops.KernelError, match="current device"):
        ops.flash_attn_window_bwd(qkv, out, dout.cpu(), lse, 1, 8, 2, 1, HD, 4)


@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", [(2, 97, 8, 2, 97, 0), (1, 256, 8, 2, 200, 4), (3, 700, 4, 4, 64, 30), (1, 3000, 8, 1, 1024, 4), (4, 513, 4, 2, 513, 0), (2, 1200, 8, 4, 20, 5)])
def test_early_rows_of_long_sequences_are_no_less_exact(B, S, nh, nkv, window, sinks):
    """The first queries of a sequence see few keys, however long it is and whatever the window: their dq alone, within what test_few_visible_keys_are_no_less_exact
    asks of whole tensors. (A query behind the first 24 of these shapes sees at least 25.)"""
    from cai_b200 import ops
    qkv, dout = _inputs(B, S, nh, nkv, 23)
    out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, window, sinks)
    dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, HD, window, sinks)
    d = _reference(qkv, dout, B, S, nh, nkv, window, sinks, HD ** -0.5)[3]
    got, want = (t.double().view(B, S, -1)[:, :24, :nh * HD] for t in (dqkv, d))
    for rows in (slice(0, 6), slice(6, 24), slice(0, 24)):
        once = (want[:, rows].to(torch.bfloat16).double() - want[:, rows]).norm()
        assert (got[:, rows] - want[:, rows]).norm() <= 1.6 * once
