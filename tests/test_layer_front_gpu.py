"""The e4m3 norm and the rotary positions of several axes against their formulas in 64 bits, and the attention half of a layer made of them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8        # half a step of bf16, of the value


# ---------------------------------------------------------------------------- norm
def _norm_inputs(rows, H, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, H, device="cuda", generator=g) * torch.exp(torch.randn(H, device="cuda", generator=g))).to(torch.bfloat16)
    r = torch.randn(rows, H, device="cuda", generator=g).to(torch.bfloat16)
    return x, r, (1 + 0.3 * torch.randn(H, device="cuda", generator=g)).to(torch.bfloat16)


def _check_norm(x, r, g, eps, got):
    h, q, s, rstd, y = got
    rows, H = x.shape
    hd = x.double() if r is None else (x.float() + r.float()).to(torch.bfloat16).double()
    assert torch.equal(h.double(), hd)
    rr = (hd.square().mean(1) + eps).rsqrt()
    # up to 64 squares a lane, five sums across a warp, eight warps, in fp32: a sum of positive terms is off by 80 roundings of 2^-24 at most
    rel = 80 * 2.0 ** -24
    assert ((rstd.double() - rr).abs() <= rel * rr).all()
    yd = hd * rr[:, None] * g.double()
    if y is not None:
        assert ((y.double() - yd).abs() <= (HALF + rel) * yd.abs()).all()
    sd = yd.view(rows, H // 128, 128).abs().amax(2) / 448
    sd = torch.where(sd > 0, sd, torch.ones_like(sd))
    assert s.shape == sd.shape and ((s.double() - sd).abs() <= (rel + 4 * 2.0 ** -24) * sd).all()
    # rounded once: half a step, 2^-4 of the value or half of the smallest step, 2^-10, from y / s; the quotient is a product with 1 / s
    z = yd / sd.repeat_interleave(128, 1)
    qd = q.double()
    assert ((qd - z).abs() <= (2.0 ** -4 + 2 * rel) * z.abs().clamp_min(2.0 ** -6)).all()
    assert (q.float().abs() <= 448).all() and (q.view(rows, H // 128, 128).float().abs().amax(2) == 448).logical_or(sd == 1).all()


@pytest.mark.parametrize("rows,H", [(1, 128), (3, 128), (7, 256), (1, 384), (5, 512), (33, 640), (256, 1024), (1777, 1408), (100, 2048), (9, 2176), (300, 4096), (13, 5120), (4, 8192),
                                    (2, 8320), (3, 16384), (5, 14336)])
@pytest.mark.parametrize("residual,keep_y", [(0, 0), (1, 1), (1, 0), (0, 1)])
def test_norm(rows, H, residual, keep_y):
    from cai_b200 import ops
    x, r, g = _norm_inputs(rows, H)
    r = r if residual else None
    got = ops.add_rmsnorm_quant(x, r, g, 1e-5, keep_y=bool(keep_y))
    assert (got[4] is not None) == bool(keep_y) and (r is not None or got[0] is x)
    _check_norm(x, r, g, 1e-5, got)


def test_norm_of_many_rows():
    from cai_b200 import ops
    x, r, g = _norm_inputs(20001, 1024, 4)
    _check_norm(x, r, g, 1e-6, ops.add_rmsnorm_quant(x, r, g, keep_y=True))


@pytest.mark.parametrize("rows,H", [(1, 128), (5, 384), (333, 1408)])
def test_norm_results_are_apart(rows, H):
    """Results share allocations: each starts on 16 bytes, ends before the next one, and is changed without the others; one that is kept keeps its values."""
    from cai_b200 import ops
    x, r, g = _norm_inputs(rows, H, 6)
    got = ops.add_rmsnorm_quant(x, r, g, keep_y=True)
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in got)
    assert all(a % 16 == 0 for a, _ in spans[:1]) and all(t.data_ptr() % 16 == 0 for t in got[:3])
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    for t in got:
        assert t.is_contiguous() and t.data_ptr() + t.numel() * t.element_size() <= t.untyped_storage().data_ptr() + t.untyped_storage().nbytes()
    want = [t.clone() for t in got]
    for i, t in enumerate(got):
        t.view(torch.uint8).fill_(0x3c)
        for k in range(i + 1, len(got)):
            assert torch.equal(got[k].view(torch.uint8), want[k].view(torch.uint8))
    h, q, s, rstd, y = ops.add_rmsnorm_quant(x, r, g, keep_y=True)
    del h, y, q
    other = [torch.full((rows, H), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(8)]
    assert torch.equal(s, want[2]) and torch.equal(rstd, want[3]) and len(other) == 8


def test_norm_of_no_rows():
    from cai_b200 import ops
    x, g = torch.zeros(0, 256, device="cuda", dtype=torch.bfloat16), torch.ones(256, device="cuda", dtype=torch.bfloat16)
    for r, keep in ((x, True), (None, False)):
        h, q, s, rstd, y = ops.add_rmsnorm_quant(x, r, g, keep_y=keep)
        assert h.shape == (0, 256) and q.shape == (0, 256) and s.shape == (0, 2) and rstd.shape == (0,) and (y is None or y.shape == (0, 256))


def test_results_are_freed_and_handed_to_streams():
    """What a call returns is freed when the last of what shares its memory goes, and may be recorded on another stream."""
    from cai_b200 import ops
    x, r, g = _norm_inputs(4096, 1024, 2)
    ops.add_rmsnorm_quant(x, r, g, keep_y=True)
    torch.cuda.synchronize()
    before, side = torch.cuda.memory_allocated(), torch.cuda.Stream()
    got = ops.add_rmsnorm_quant(x, r, g, keep_y=True)
    want = got[2].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept = got[2].clone()
    got[2].record_stream(side)
    assert torch.cuda.memory_allocated() > before
    del got
    torch.cuda.synchronize()
    assert torch.equal(kept, want)
    del kept, want
    torch.cuda.synchronize()
    torch.zeros(1, device="cuda")          # the allocator looks at what has been recorded
    assert torch.cuda.memory_allocated() <= before


def test_offsets_beyond_32_bits():
    from cai_b200 import ops
    rows, H = 300 * 1024, 8192
    assert rows * H > 1 << 31
    x, r, g = _norm_inputs(1024, H, 12)
    X, R = x.repeat(300, 1), r.repeat(300, 1)
    want, got = ops.add_rmsnorm_quant(x, r, g, keep_y=True), ops.add_rmsnorm_quant(X, R, g, keep_y=True)
    for a, b in zip(want, got):
        assert torch.equal(a.view(torch.uint8), b[-1024:].view(torch.uint8)) and torch.equal(a.view(torch.uint8), b[150 * 1024:151 * 1024].view(torch.uint8))
    del X, R, got, want
    T, nh, nkv = 384 * 1024, 40, 4
    qkv = torch.randn(4096, 48 * 128, device="cuda").to(torch.bfloat16)
    pos, freqs = torch.randint(0, 5000, (2, 4096), device="cuda", dtype=torch.int32), ops.rope_freqs(128)
    big = qkv.repeat(T // 4096, 1)
    assert big.numel() > 1 << 31
    ops.rope_apply_axes_(big, freqs, pos.repeat(1, T // 4096), nh, nkv, 128, (32, 32))
    ops.rope_apply_axes_(qkv, freqs, pos, nh, nkv, 128, (32, 32))
    assert torch.equal(big[-4096:], qkv)


def test_norm_of_views():
    """Rows with pitches of their own, a residual that is one row for all, rows that start in the middle of a buffer of NaN."""
    from cai_b200 import ops
    x, r, g = _norm_inputs(50, 384, 1)
    big = torch.full((60, 384 + 40), float("nan"), device="cuda", dtype=torch.bfloat16)
    big[5:55, 16:400] = x
    v = big[5:55, 16:400]
    _check_norm(v, r[:1].expand(50, 384), g, 1e-6, ops.add_rmsnorm_quant(v, r[:1].expand(50, 384), g, keep_y=True))
    _check_norm(v[::2], r[::2], g, 1e-6, ops.add_rmsnorm_quant(v[::2], r[::2], g))
    one = ops.add_rmsnorm_quant(v[:1], None, g)
    _check_norm(v[:1], None, g, 1e-6, one)


def test_norm_of_zeros_and_of_what_is_not_finite():
    """A row of zeros: scale 1, as the quantiser of its own gives. A row that is not finite spoils itself alone."""
    from cai_b200 import ops
    x, _, g = _norm_inputs(6, 256, 2)
    want = ops.add_rmsnorm_quant(x, None, g, keep_y=True)
    x[1] = 0
    x[3, 5] = float("nan")
    x[4, 200] = float("inf")
    h, q, s, rstd, y = ops.add_rmsnorm_quant(x, None, g, keep_y=True)
    assert (q[1].float() == 0).all() and (s[1] == 1).all() and abs(rstd[1].item() - 1e3) < 1e-2
    assert q[3].float().isnan().all() and y[3].isnan().all() and rstd[4] == 0
    for got, w in zip((q, s, rstd, y), want[1:]):
        for row in (0, 2, 5):
            assert torch.equal(got[row].float(), w[row].float())
    assert ops.add_rmsnorm_quant(x[:0], None, g, keep_y=True)[1].shape == (0, 256)


def test_norm_of_very_small_rows():
    """Blocks whose largest magnitude is 2^-120 or less beside ordinary ones: no scale whose reciprocal leaves fp32, no NaN."""
    from cai_b200 import ops
    x = torch.ones(3, 512, device="cuda", dtype=torch.bfloat16)
    g = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    g[128:256] = 2.0 ** -125
    g[256:384] = 0
    g[300] = -2.0 ** -133
    h, q, s, rstd, y = ops.add_rmsnorm_quant(x, None, g, keep_y=True)
    assert torch.isfinite(q.float()).all() and torch.isfinite(s).all() and torch.isfinite(1 / s).all()
    back = q.float() * s.repeat_interleave(128, 1)
    # (1 + eps)^(-1/2) is the block's largest and its only value: 448 scales, within their rounding; y rounds it to 1
    assert ((back[:, :128] - rstd[:, None]).abs() <= 2.0 ** -22).all() and (y[:, :128] == 1).all() and (back[:, 128:384].abs() <= 2.0 ** -120).all()


def test_norm_gives_what_its_parts_give():
    """Against the norm and the quantiser of their own: the same stream and statistics, e4m3 numbers at most a step apart (their y is rounded in between)."""
    from cai_b200 import ops
    x, r, g = _norm_inputs(123, 512, 3)
    h, q, s, rstd, y = ops.add_rmsnorm_quant(x, r, g, keep_y=True)
    y2, rstd2 = ops.rmsnorm_fwd(h, g)
    q2, s2 = ops.quant_rows_1x128(y2)
    assert torch.allclose(rstd, rstd2, rtol=1e-5) and (y.float() - y2.float()).abs().max() <= HALF * 2 * y.float().abs().max()
    assert ((s - s2).abs() <= 2 * HALF * s).all()
    a, b = q.float() * s.repeat_interleave(128, 1), q2.float() * s2.repeat_interleave(128, 1)
    assert ((a - b).abs() <= 2.0 ** -3 * a.abs().clamp_min(2.0 ** -6 * s.amax().item()) * 1.05).all()


def test_norm_gradient():
    """rmsnorm_bwd on h with the gradient that comes past the norm: that of x and of the residual; against the formula and differences in 64 bits."""
    from cai_b200 import ops
    x, r, g = _norm_inputs(40, 256, 5)
    h, q, s, rstd, y = ops.add_rmsnorm_quant(x, r, g, 1e-6, keep_y=True)
    dy, dh = (torch.randn(40, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)).to(torch.bfloat16) for k in (1, 2))
    dx, dg = ops.rmsnorm_bwd(h, g, rstd, dy, dx=dh.clone(), dx_accumulate=True)

    def loss(hh, gg):
        return (hh * (hh.square().mean(1, keepdim=True) + 1e-6).rsqrt() * gg * dy.double()).sum() + (hh * dh.double()).sum()
    hd, gd = h.double().requires_grad_(True), g.double().requires_grad_(True)
    loss(hd, gd).backward()
    tol = HALF * hd.grad.abs() + 2.0 ** -16 * (dy.double() * gd).abs().amax(1, keepdim=True) * rstd.double()[:, None] + 2.0 ** -16 * dh.double().abs()
    assert ((dx.double() - hd.grad).abs() <= tol).all()
    assert ((dg.double() - gd.grad).abs() <= 2.0 ** -16 * (dy.double() * h.double() * rstd.double()[:, None]).abs().sum(0)).all()
    u = torch.randn(40, 256, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(3))
    slope = (loss(h.double() + 1e-6 * u, g.double()) - loss(h.double() - 1e-6 * u, g.double())) / 2e-6
    assert (slope - (dx.double() * u).sum()).abs() <= 4 * tol.detach().norm() + 1e-6 * slope.abs()


# ---------------------------------------------------------------------------- rotary positions
def _axis(half, sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    m = len(sections)
    return [i % m if i // m < sections[i % m] else 0 for i in range(half)]


def _rope(qkv, freqs, pos, nh, nkv, hd, sections, interleaved, inverse):
    """The turned q and k heads in 64 bits, and how far they may be off: half a step, and two products and angles in fp32."""
    half = hd // 2
    x = qkv[:, :(nh + nkv) * hd].double().view(qkv.shape[0], nh + nkv, 2, half)
    angle = pos[_axis(half, sections, interleaved)].t().double() * freqs
    c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if inverse else 1)
    a, b = x[:, :, 0], x[:, :, 1]
    y = torch.stack([a * c - b * s, b * c + a * s], 2)
    return y.flatten(1), (HALF * y.abs() + 2.0 ** -21 * (a.abs() + b.abs())[:, :, None]).flatten(1)


ROPES = [(1, 1, 1, 128, (64,), 0), (2, 2, 1, 128, (22, 21, 21), 1), (17, 4, 2, 128, (16, 24, 24), 0), (300, 9, 3, 128, (24, 20, 20), 1), (1000, 32, 8, 128, (32, 32), 0), (33, 3, 3, 64, (8, 8, 8, 8), 1),
         (5, 2, 2, 16, (4, 2, 2), 0), (70, 5, 1, 256, (128, 0, 0), 0), (9, 1, 0, 96, (0, 48), 0), (4097, 2, 1, 80, (14, 13, 13), 1), (3, 50, 10, 256, (43, 43, 42), 0)]


@pytest.mark.parametrize("T,nh,nkv,hd,sections,interleaved", ROPES)
@pytest.mark.parametrize("span", [50, 2 ** 31 - 1])
def test_rope_axes(T, nh, nkv, hd, sections, interleaved, span):
    from cai_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, device="cuda", generator=g).to(torch.bfloat16)
    pos = torch.randint(-span, span, (len(sections), T), device="cuda", generator=g, dtype=torch.int32)
    freqs = ops.rope_freqs(hd)
    for inverse in (False, True):
        x = qkv.clone()
        assert ops.rope_apply_axes_(x, freqs, pos, nh, nkv, hd, sections, interleaved=bool(interleaved), inverse=inverse) is x
        want, tol = _rope(qkv, freqs, pos, nh, nkv, hd, sections, interleaved, inverse)
        n = (nh + nkv) * hd
        # the reference's own angle of 2^31 radians is off by 2^-22
        assert ((x[:, :n].double() - want).abs() <= tol + (2.0 ** -20 if span > 2 ** 20 else 0) * 8).all()
        assert torch.equal(x[:, n:], qkv[:, n:])


def test_rope_axes_of_views():
    from cai_b200 import ops
    T, nh, nkv, hd, sections = 37, 2, 1, 128, (16, 24, 24)
    big = torch.randn(T + 4, 4 * hd + 32, device="cuda").to(torch.bfloat16)
    kept = big.clone()
    pos = torch.randint(0, 999, (3, 2 * T), device="cuda", dtype=torch.int32)
    v, p, freqs = big[2:2 + T, 16:16 + 4 * hd], pos[:, 5:5 + T], ops.rope_freqs(hd, 1e6)
    want, tol = _rope(v, freqs, p, nh, nkv, hd, sections, 0, False)
    ops.rope_apply_axes_(v, freqs, p, nh, nkv, hd, sections)
    assert ((v[:, :3 * hd].double() - want).abs() <= tol).all()
    big[2:2 + T, 16:16 + 3 * hd] = kept[2:2 + T, 16:16 + 3 * hd]
    assert torch.equal(big, kept)


def test_rope_axes_of_one_row_of_positions_for_all():
    from cai_b200 import ops
    qkv = torch.randn(9, 512, device="cuda").to(torch.bfloat16)
    pos = torch.arange(100, 109, device="cuda", dtype=torch.int32)[None].expand(3, 9)
    a, b = qkv.clone(), qkv.clone()
    ops.rope_apply_axes_(a, ops.rope_freqs(128), pos, 2, 1, 128, [16, 24, 24])
    ops.rope_apply_axes_(b, ops.rope_freqs(128), pos[:1].contiguous(), 2, 1, 128, [64])
    assert torch.equal(a, b) and not torch.equal(a, qkv)


def test_rope_axes_is_the_one_axis_rotation():
    """One axis with position t mod seq: what rope_apply_ does with its table, as near as that table's angles are."""
    from cai_b200 import ops
    T, seq, nh, nkv, hd = 96, 48, 4, 2, 128
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, device="cuda").to(torch.bfloat16)
    a, b = qkv.clone(), qkv.clone()
    ops.rope_apply_(a, ops.rope_table(seq, hd), seq, nh, nkv, hd)
    ops.rope_apply_axes_(b, ops.rope_freqs(hd), (torch.arange(T, device="cuda", dtype=torch.int32) % seq)[None], nh, nkv, hd, (64,))
    assert ((a.float() - b.float()).abs() <= 2 * HALF * a.float().abs() + 1e-4).all()


def test_rope_axes_gradient_is_the_inverse_turn():
    """The turn is linear: the gradient of sum(w * turn(x)) is w turned back; against the differences, which are exact for a linear function."""
    from cai_b200 import ops
    T, nh, nkv, hd, sections = 20, 2, 1, 128, (22, 21, 21)
    g = torch.Generator(device="cuda").manual_seed(0)
    w, u = (torch.randn(T, 4 * hd, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    pos = torch.randint(0, 5000, (3, T), device="cuda", generator=g, dtype=torch.int32)
    freqs, n = ops.rope_freqs(hd), 3 * hd
    grad = ops.rope_apply_axes_(w.clone(), freqs, pos, nh, nkv, hd, sections, inverse=True)
    turned, _ = _rope(u, freqs, pos, nh, nkv, hd, sections, 0, False)
    slope = (turned * w[:, :n].double()).sum()
    _, tol = _rope(w, freqs, pos, nh, nkv, hd, sections, 0, True)
    assert (slope - (grad[:, :n].double() * u[:, :n].double()).sum()).abs() <= 4 * (tol * u[:, :n].double().abs()).norm()


def test_rope_axes_of_no_tokens():
    from cai_b200 import ops
    x = torch.zeros(0, 512, device="cuda", dtype=torch.bfloat16)
    assert ops.rope_apply_axes_(x, ops.rope_freqs(128), torch.zeros(2, 0, device="cuda", dtype=torch.int32), 2, 1, 128, (32, 32)) is x


def test_front_calls_refuse_tensors_elsewhere():
    from cai_b200 import ops
    x, r, g = _norm_inputs(4, 128)
    with pytest.raises(ops.KernelError, match="current device"):
        ops.add_rmsnorm_quant(x, r.cpu(), g)
    with pytest.raises(ops.KernelError, match="current device"):
        ops.rope_apply_axes_(torch.zeros(2, 512, device="cuda", dtype=torch.bfloat16), ops.rope_freqs(128, device="cpu"), torch.zeros(1, 2, device="cuda", dtype=torch.int32), 2, 1, 128, (64,))


# ---------------------------------------------------------------------------- together
def _half_layer(B, S, nh, nkv, H, window, sinks, sections, seed=0):
    from cai_b200 import ops
    hd, g = 128, torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(torch.bfloat16)
    T, cols = B * S, (nh + 2 * nkv) * hd
    p = dict(x=normal(T, H), branch=normal(T, H, scale=0.5), gain=(1 + 0.1 * torch.randn(H, device="cuda", generator=g)).to(torch.bfloat16),
             wqkv=normal(cols, H, scale=H ** -0.5), wo=normal(H, nh * hd, scale=(nh * hd) ** -0.5), dy=normal(T, H), freqs=ops.rope_freqs(hd),
             pos=torch.randint(0, 3000, (len(sections), T), device="cuda", generator=g, dtype=torch.int32))
    p["wq"], p["ws"] = ops.quant_blocks_128x128(p["wqkv"])

    def step():
        """The stream after the attention half, the gradients of its two inputs, of the gain and of the projections."""
        h, q, s, rstd, y = ops.add_rmsnorm_quant(p["x"], p["branch"], p["gain"], 1e-6, keep_y=True)
        qkv = ops.gemm_fp8(q, s, p["wq"], p["ws"])
        ops.rope_apply_axes_(qkv, p["freqs"], p["pos"], nh, nkv, hd, sections)
        out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, hd, window, sinks)
        z = ops.gemm(out, p["wo"], residual=h)
        dout = ops.gemm(p["dy"], p["wo"], trans_b=True)
        dwo = ops.gemm(p["dy"], out, trans_a=True, trans_b=True, out_dtype=torch.float32)
        dqkv = ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, hd, window, sinks)
        ops.rope_apply_axes_(dqkv, p["freqs"], p["pos"], nh, nkv, hd, sections, inverse=True)
        dwqkv = ops.gemm(dqkv, y, trans_a=True, trans_b=True, out_dtype=torch.float32)
        dn = ops.gemm(dqkv, p["wqkv"], trans_b=True)
        dx, dg = ops.rmsnorm_bwd(h, p["gain"], rstd, dn, dx=p["dy"].clone(), dx_accumulate=True)
        return dict(z=z, dx=dx, dg=dg, dwqkv=dwqkv, dwo=dwo)
    return p, step


def _half_layer_reference(p, B, S, nh, nkv, window, sinks, sections):
    """The same in 64 bits: the e4m3 operands are quantised by their definitions (their gradients are those of what was quantised)."""
    from cai_b200 import ops
    hd, T, H = 128, B * S, p["x"].shape[1]
    h = (p["x"].float() + p["branch"].float()).to(torch.bfloat16).double().requires_grad_(True)
    gain, w, wo = (p[k].double().requires_grad_(True) for k in ("gain", "wqkv", "wo"))
    n = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * gain
    with torch.no_grad():
        s = n.view(T, H // 128, 128).abs().amax(2) / 448
        nq = ((n / s.repeat_interleave(128, 1)).float().to(torch.float8_e4m3fn).double() * s.repeat_interleave(128, 1))
        wd = p["wq"].double() * p["ws"].double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:w.shape[0], :H]
    qkv = (n + (nq - n).detach()) @ wd.t() + n.detach() @ (w - w.detach()).t() + (n - n.detach()) @ (w - wd).detach().t()
    x = qkv.view(T, nh + 2 * nkv, 2, 64)
    angle = p["pos"][_axis(64, sections, 0)].t().double() * p["freqs"]
    c, sn = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[:, :nh + nkv, 0], x[:, :nh + nkv, 1]
    turned = torch.cat([torch.stack([a * c - b * sn, b * c + a * sn], 2), x[:, nh + nkv:]], 1).reshape(B, S, nh + 2 * nkv, hd).transpose(1, 2)
    rep = nh // nkv
    q, k, v = turned[:, :nh], turned[:, nh:nh + nkv].repeat_interleave(rep, 1), turned[:, nh + nkv:].repeat_interleave(rep, 1)
    i, j = torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None]
    att = (q @ k.transpose(2, 3) * hd ** -0.5).masked_fill(~((j <= i) & ((j > i - window) | (j < sinks))), -math.inf)
    o = (torch.softmax(att, -1) @ v).transpose(1, 2).reshape(T, nh * hd)
    z = h + o @ wo.t()
    z.backward(p["dy"].double())
    return dict(z=z.detach(), dx=h.grad, dg=gain.grad, dwqkv=w.grad, dwo=wo.grad)


@pytest.mark.parametrize("B,S,nh,nkv,H,window,sinks,sections", [(2, 160, 2, 1, 256, 50, 3, (22, 21, 21)), (1, 700, 6, 2, 640, 128, 1, (64,)), (3, 33, 4, 4, 384, 8, 20, (32, 32))])
def test_the_attention_half_of_a_layer(B, S, nh, nkv, H, window, sinks, sections):
    """Forward and backward, as a training program calls it. Between input and result lie some ten roundings to bf16, half a step each and
    independent of one another; as norms they add up to less than sqrt(10 / 3) half steps, twice that is allowed."""
    p, step = _half_layer(B, S, nh, nkv, H, window, sinks, sections)
    got, want = step(), _half_layer_reference(p, B, S, nh, nkv, window, sinks, sections)
    for k, w in want.items():
        assert (got[k].double() - w).norm() <= 2 * math.sqrt(10 / 3) * HALF * w.norm(), k


def test_the_attention_half_captured_beside_an_eager_one():
    """The step in a graph while an eager one runs on another stream and its results live on: the same bits from both."""
    p, step = _half_layer(2, 300, 4, 2, 512, 64, 4, (16, 24, 24))
    _, other = _half_layer(1, 200, 2, 1, 256, 100, 0, (64,), seed=1)
    want, want_other = step(), other()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    side = torch.cuda.Stream()
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            beside = other()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(held[k], want[k]) and torch.equal(beside[k], want_other[k]), k
