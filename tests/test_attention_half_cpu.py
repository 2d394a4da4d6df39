"""Windowed attention, rotary positions of several axes and the e4m3 norm, as far as no GPU is needed: which tiles the CTAs of windowed attention take, and what
the calls refuse."""
import ctypes

import pytest
import torch

T = 128


def _seen(i, j, window, sinks):
    return j <= i and (j > i - window or j < sinks)


def _tile_pairs(S, window, sinks):
    """(query tile, key tile) of every pair of tiles in which some query sees some key."""
    n = (S + T - 1) // T
    found = set()
    for i in range(n):
        for j in range(i + 1):
            q_last, k_first, k_last = min(S, (i + 1) * T) - 1, j * T, min(S, (j + 1) * T) - 1
            # the nearest pair decides for the window, the first key for the sinks
            nearest = max(i * T, k_first) - min(k_last, i * T) if i > j else 0
            if nearest < window or k_first < sinks:
                assert k_first <= q_last
                found.add((i, j))
    return found


SHAPES = [(1, 1, 1, 1, 1, 0), (2, 128, 2, 1, 64, 4), (3, 129, 4, 2, 1, 0), (1, 1000, 9, 3, 200, 0), (1, 333, 8, 1, 512, 1), (4, 4096, 16, 8, 1024, 4),
          (1, 8192, 4, 1, 128, 130), (1, 8192, 8, 8, 2, 512), (2, 2000, 6, 2, 129, 127), (1, 5000, 8, 1, 257, 5000), (7, 640, 3, 3, 128, 128),
          (1, 16384, 2, 1, 300, 1), (1, 3000, 16, 2, 127, 300)]


def _taken(call, S, window, sinks, i):
    """(number, keys that the products take) of what query tile i takes."""
    found = (ctypes.c_int * 8192)()
    n = call(S, window, sinks, i, found, 4096)
    assert 0 < n <= 4096
    return [(found[2 * k], found[2 * k + 1]) for k in range(n)]


@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", SHAPES)
def test_dq_takes_every_key_tile_once(B, S, nh, nkv, window, sinks):
    from cai_b200.ops import lib
    got = set()
    for i in range((S + T - 1) // T):
        tiles = _taken(lib().cai_flash_attn_window_keys, S, window, sinks, i)
        numbers = [t for t, _ in tiles]
        assert numbers == sorted(set(numbers)) and numbers[-1] == i, "in order, the diagonal last"
        for t, width in tiles:
            # all keys, or of a tile that is behind every window of the query tile the sinks, 16 at a time
            assert width == T or (width % 16 == 0 and sinks <= t * T + width < sinks + 16 and (t + 1) * T - 1 <= i * T - window)
        got |= {(i, t) for t in numbers}
    assert got == _tile_pairs(S, window, sinks)


@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", SHAPES)
def test_forward_takes_every_block_of_keys_once(B, S, nh, nkv, window, sinks):
    from cai_b200.ops import lib
    K = 64
    for i in range((S + T - 1) // T):
        blocks = _taken(lib().cai_flash_attn_window_blocks, S, window, sinks, i)
        numbers = [k for k, _ in blocks]
        assert numbers == sorted(set(numbers))
        q_first, q_last = i * T, min(S, (i + 1) * T) - 1
        want = [k for k in range(q_last // K + 1) if min(k * K + K - 1, q_first) > q_first - window or k * K < sinks]
        assert numbers == want
        for k, width in blocks:
            assert width == K or (width % 16 == 0 and sinks <= k * K + width < sinks + 16 and (k + 1) * K - 1 <= q_first - window)


@pytest.mark.parametrize("B,S,nh,ctas", [(1, 1, 1, 1), (3, 300, 5, 45), (4, 4096, 16, 296), (1, 2000, 32, 296), (2, 9000, 3, 296), (7, 130, 9, 17), (1, 32768, 4, 296)])
def test_forward_items_are_taken_once(B, S, nh, ctas):
    from cai_b200.ops import lib
    seen, most, least = set(), 0, 1 << 30
    for cta in range(ctas):
        found = (ctypes.c_int * 30000)()
        n = lib().cai_flash_attn_window_items(B, S, nh, ctas, cta, found, 10000)
        most, least = max(most, n), min(least, n)
        for k in range(n):
            t = tuple(found[3 * k:3 * k + 3])
            assert t not in seen
            seen.add(t)
    assert seen == {(i, h, b) for i in range((S + T - 1) // T) for h in range(nh) for b in range(B)}
    assert most - least <= 1


@pytest.mark.parametrize("sms", [148, 8, 1])
@pytest.mark.parametrize("B,S,nh,nkv,window,sinks", SHAPES)
def test_backward_parts_cover_every_sum_once(B, S, nh, nkv, window, sinks, sms):
    """Every (batch, query head, query tile, key tile) lies in one CTA's part; parts of one key tile have scratch of their own, or the tile has one part."""
    from cai_b200.ops import lib
    n = lib().cai_flash_attn_window_walk(B, S, nh, nkv, window, sinks, sms, None, 0)
    parts = (ctypes.c_int * (8 * n))()
    assert lib().cai_flash_attn_window_walk(B, S, nh, nkv, window, sinks, sms, parts, n) == n
    seen, slots, of_tile = set(), set(), {}
    for c in range(n):
        j, b, g, h0, heads, q0, tiles, slot = parts[8 * c:8 * c + 8]
        assert 0 <= b < B and 0 <= g < nkv and heads >= 1 and g * (nh // nkv) <= h0 and h0 + heads <= (g + 1) * (nh // nkv)
        if tiles <= 0:
            continue
        assert 0 <= j <= q0 and (q0 + tiles - 1) * T < S
        of_tile.setdefault((b, g, j), []).append(slot)
        assert slot < 0 or slot not in slots
        slots.add(slot)
        for h in range(h0, h0 + heads):
            for i in range(q0, q0 + tiles):
                assert (b, h, i, j) not in seen
                seen.add((b, h, i, j))
    want = _tile_pairs(S, window, sinks)
    assert seen == {(b, h, i, j) for b in range(B) for h in range(nh) for i, j in want}
    assert len(of_tile) == B * nkv * ((S + T - 1) // T), "every key tile's rows are written"
    for s in of_tile.values():
        assert len(s) == 1 and s[0] == -1 or min(s) >= 0
    if sms == 148:
        most = lib().cai_flash_attn_window_bwd_scratch(B, S, nh, nkv, window, sinks)
        assert max(slots) * 131072 + 131072 <= most or max(slots) < 0


def test_parts_of_sink_tiles_are_no_longer_than_a_share():
    """One kv head of a very long sequence: the first tile's 256 query tiles are cut into parts, the scratch stays that of about one part a SM."""
    from cai_b200.ops import lib
    B, S, nh, nkv, window, sinks = 1, 32768, 4, 1, 2048, 130
    n = lib().cai_flash_attn_window_walk(B, S, nh, nkv, window, sinks, 148, None, 0)
    parts = (ctypes.c_int * (8 * n))()
    lib().cai_flash_attn_window_walk(B, S, nh, nkv, window, sinks, 148, parts, n)
    steps = [parts[8 * c + 4] * max(0, parts[8 * c + 6]) for c in range(n)]
    assert max(steps) <= 2 * 4 * (2048 // T + 1)
    assert lib().cai_flash_attn_window_bwd_scratch(B, S, nh, nkv, window, sinks) <= 2 * 148 * 2 * 131072


# ---------------------------------------------------------------------------- refusals
P = 1 << 20      # an address that no refused call looks at


def _window(name, **change):
    a = dict(qkv=P, ld=512, out=P, lse=P, dout=P, delta=P, dqkv=P, ldq=512, scratch=P, B=1, S=256, nh=2, nkv=1, hd=128, scale=0.1, window=64, sinks=4, stream=0)
    a.update(change)
    if name == "fwd":
        order = ("qkv", "ld", "out", "lse", "B", "S", "nh", "nkv", "hd", "scale", "window", "sinks", "stream")
    else:
        order = ("qkv", "ld", "out", "dout", "lse", "delta", "dqkv", "ldq", "scratch", "B", "S", "nh", "nkv", "hd", "scale", "window", "sinks", "stream")
    return [a[k] for k in order]


BAD_WINDOW = [dict(hd=64), dict(nh=3, nkv=2, ld=1024, ldq=1024), dict(nkv=0), dict(nh=0), dict(window=0), dict(window=-5), dict(sinks=-1), dict(ld=504, ldq=504),
              dict(ld=516, ldq=516), dict(qkv=P + 8), dict(out=P + 8), dict(scale=0.0), dict(scale=-0.1), dict(scale=float('inf')), dict(scale=float('nan')), dict(B=-1), dict(S=-1), dict(B=70000), dict(B=60000, S=60000)]


@pytest.mark.parametrize("change", BAD_WINDOW, ids=str)
@pytest.mark.parametrize("name", ["fwd", "bwd"])
def test_window_launchers_refuse(name, change):
    from cai_b200.ops import KernelError, calls, check
    f = getattr(calls(), f"cai_flash_attn_window_{name}")
    with pytest.raises(KernelError, match="flash_attn_window"):
        check(f(*_window(name, **change)), "flash_attn_window")


@pytest.mark.parametrize("change", [dict(dout=P + 2), dict(dqkv=P + 4), dict(ldq=500), dict(scratch=P + 4)], ids=str)
def test_window_bwd_launcher_refuses(change):
    from cai_b200.ops import KernelError, calls, check
    with pytest.raises(KernelError, match="flash_attn_window_bwd"):
        check(calls().cai_flash_attn_window_bwd(*_window("bwd", **change)), "flash_attn_window")


@pytest.mark.parametrize("name", ["fwd", "bwd"])
@pytest.mark.parametrize("change", [dict(B=0), dict(S=0)], ids=str)
def test_window_launchers_do_nothing_for_no_rows(name, change):
    from cai_b200.ops import calls
    assert getattr(calls(), f"cai_flash_attn_window_{name}")(*_window(name, **change)) == 0


def test_window_calls_refuse_tensors_that_do_not_fit():
    from cai_b200 import ops
    B, S, nh, nkv = 2, 10, 2, 1
    qkv = torch.zeros(B * S, 4 * 128, dtype=torch.bfloat16)
    out, lse = torch.zeros(B * S, 256, dtype=torch.bfloat16), torch.zeros(B, nh, S)
    for bad in (qkv.float(), qkv[1:], qkv[:, 1:], qkv.t(), qkv.view(-1).as_strided((B * S, 512), (256, 1))):
        with pytest.raises(ops.KernelError, match="flash_attn_window_fwd"):
            ops.flash_attn_window_fwd(bad, B, S, nh, nkv, 128, 4)
        with pytest.raises(ops.KernelError, match="flash_attn_window_bwd"):
            ops.flash_attn_window_bwd(bad, out, out, lse, B, S, nh, nkv, 128, 4)
    for o, d, l in ((out.float(), out, lse), (out, out[:, :128], lse), (out, out, lse.double()), (out, out, lse[:, :1]), (out, out.t().contiguous().t(), lse)):
        with pytest.raises(ops.KernelError, match="flash_attn_window_bwd"):
            ops.flash_attn_window_bwd(qkv, o, d, l, B, S, nh, nkv, 128, 4)


def test_window_bwd_refuses_workspaces_and_gradients_over_other_arguments():
    """lse's place for delta would give no error and wrong gradients: every CTA reads lse while delta is written."""
    from cai_b200 import ops
    B, S, nh, nkv = 2, 300, 2, 1
    bf16, n = torch.bfloat16, 600
    qkv, out, dout, lse = torch.zeros(n, 512, dtype=bf16), torch.zeros(n, 256, dtype=bf16), torch.zeros(n, 256, dtype=bf16), torch.zeros(B, nh, S)
    dqkv, delta = torch.zeros(n, 512, dtype=bf16), torch.zeros(B, nh, S)
    need = ops.flash_attn_window_bwd_scratch(B, S, nh, nkv, 40, 3)
    assert need > 0
    both = torch.zeros(need + 4 * B * nh * S, dtype=torch.uint8)

    def of(t, dtype=torch.float32):
        return t.view(-1).view(dtype)
    cases = [dict(delta=lse), dict(delta=of(qkv)), dict(delta=of(out)), dict(delta=of(dout)[-B * nh * S:]), dict(dqkv=dqkv, delta=of(dqkv)),
             dict(scratch=both[4 * B * nh * S - 16:], delta=both[:4 * B * nh * S].view(torch.float32))]
    for change in cases:
        with pytest.raises(ops.KernelError, match="flash_attn_window_bwd: a workspace shares memory"):
            ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, 128, 40, 3, **change)
    wide = torch.zeros(n * 512, dtype=bf16)
    with pytest.raises(ops.KernelError, match="flash_attn_window_bwd: dqkv shares memory"):
        ops.flash_attn_window_bwd(qkv, out, dout, of(wide)[:B * nh * S].view(B, nh, S), B, S, nh, nkv, 128, 40, 3, dqkv=wide.view(n, 512))
    # beside one another they are taken: what is refused is the device
    for change in (dict(delta=delta, dqkv=dqkv), dict(scratch=both[4 * B * nh * S:], delta=both[:4 * B * nh * S].view(torch.float32))):
        with pytest.raises(ops.KernelError, match="current device"):
            ops.flash_attn_window_bwd(qkv, out, dout, lse, B, S, nh, nkv, 128, 40, 3, **change)


def test_scratch_of_a_window_wider_than_any_sequence():
    from cai_b200 import ops
    want = ops.flash_attn_window_bwd_scratch(1, 4000, 1, 1, 4000, 4000)
    assert want > 0
    for window, sinks in ((2 ** 31, 0), (2 ** 32, 2 ** 32 + 1), (2 ** 40, 2 ** 62)):
        assert ops.flash_attn_window_bwd_scratch(1, 4000, 1, 1, window, sinks) == want


def _rope(**change):
    a = dict(qkv=P, freqs=P, pos=P, ldp=10, T=10, nh=2, nkv=1, hd=128, ld=512, axes=3, n0=16, n1=24, n2=24, n3=0, interleaved=0, inverse=0, stream=0)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [dict(hd=120), dict(hd=272), dict(hd=0), dict(axes=0), dict(axes=5), dict(n0=15), dict(n3=1, n0=15), dict(n0=-8, n1=48), dict(ld=380),
                                    dict(ld=376), dict(qkv=P + 2), dict(ldp=-1), dict(T=-1), dict(interleaved=1)], ids=str)
def test_rope_launcher_refuses(change):
    from cai_b200.ops import KernelError, calls, check
    with pytest.raises(KernelError, match="rope_apply_axes"):
        check(calls().cai_rope_apply_axes(*_rope(**change)), "rope")


def test_rope_call_refuses_tensors_that_do_not_fit():
    from cai_b200 import ops
    qkv, freqs, pos = torch.zeros(10, 512, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.float64), torch.zeros(3, 10, dtype=torch.int32)
    good = dict(qkv=qkv, freqs=freqs, pos=pos, nh=2, nkv=1, hd=128, sections=(16, 24, 24))
    for change in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :256]), dict(qkv=qkv.t()), dict(qkv=qkv[:, ::2]), dict(freqs=freqs.float()), dict(freqs=freqs[:32]), dict(pos=pos.long()),
                   dict(pos=pos[:2]), dict(pos=pos[:, :9]), dict(pos=torch.zeros(10, 3, dtype=torch.int32).t()), dict(sections=()), dict(sections=(16, 16, 16, 8, 8))):
        with pytest.raises(ops.KernelError, match="rope_apply_axes_"):
            ops.rope_apply_axes_(**{**good, **change})


def _norm(**change):
    a = dict(x=P, ldx=256, residual=P, ldr=256, g=P, h=P, y=P, q=P, scale=P, rstd=P, rows=4, H=256, eps=1e-6, stream=0)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [dict(H=192), dict(H=16512), dict(H=0), dict(rows=-1), dict(ldx=252), dict(ldr=260), dict(x=P + 2), dict(residual=P + 8), dict(g=P + 8),
                                    dict(h=P + 8), dict(y=P + 4), dict(q=P + 1)], ids=str)
def test_norm_launcher_refuses(change):
    from cai_b200.ops import KernelError, calls, check
    with pytest.raises(KernelError, match="add_rmsnorm_quant"):
        check(calls().cai_add_rmsnorm_quant(*_norm(**change)), "norm")


def test_norm_call_refuses_tensors_that_do_not_fit():
    from cai_b200 import ops
    x, g = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256, dtype=torch.bfloat16)
    for a in ((x.float(), None, g), (x, None, g.float()), (x, None, g[:128]), (x, x[:2], g), (x, x.float(), g), (x[:, ::2], None, g[:128]), (x.view(2, 2, 256), None, g),
              (x, torch.zeros(256, 4, dtype=torch.bfloat16).t(), g)):
        with pytest.raises(ops.KernelError, match="add_rmsnorm_quant"):
            ops.add_rmsnorm_quant(*a)


def test_arguments_that_are_no_tensors_or_numbers():
    from cai_b200 import ops
    qkv = torch.zeros(4, 512, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError, match="tensor"):
        ops.flash_attn_window_fwd([1.0], 1, 4, 2, 1, 128, 4)
    with pytest.raises(ops.KernelError, match="tensor"):
        ops.add_rmsnorm_quant(qkv, qkv, None)
    with pytest.raises(TypeError):
        ops.flash_attn_window_fwd(qkv, 1, "4", 2, 1, 128, 4)
    with pytest.raises(TypeError):
        ops.rope_apply_axes_(qkv, torch.zeros(64, dtype=torch.float64), torch.zeros(1, 4, dtype=torch.int32), 2, 1, 128, 64)
    with pytest.raises(ops.KernelError, match="out of range"):
        ops.flash_attn_window_fwd(qkv, 1, 2 ** 40, 2, 1, 128, 4)


def test_tensors_of_the_host_are_refused():
    from cai_b200 import ops
    x = torch.zeros(4, 512, dtype=torch.bfloat16)
    for call in (lambda: ops.add_rmsnorm_quant(x, None, x[0]), lambda: ops.flash_attn_window_fwd(x, 1, 4, 2, 1, 128, 4),
                 lambda: ops.rope_apply_axes_(x, torch.zeros(64, dtype=torch.float64), torch.zeros(1, 4, dtype=torch.int32), 2, 1, 128, (64,)),
                 lambda: ops.flash_attn_window_bwd(x, x[:, :256].clone(), x[:, :256].clone(), torch.zeros(1, 2, 4), 1, 4, 2, 1, 128, 4)):
        with pytest.raises(ops.KernelError, match="current device"):
            call()


def test_a_build_without_the_extension_refuses(monkeypatch):
    from cai_b200.ops import _lib
    monkeypatch.setattr(_lib, "_native", None)
    monkeypatch.setattr(_lib, "_extension", lambda name: None)
    with pytest.raises(_lib.KernelError, match="_ops"):
        _lib.native()


def test_frequencies():
    from cai_b200 import ops
    f = ops.rope_freqs(128, 500000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (64,) and f[0] == 1.0
    assert abs(f[32].item() - 500000.0 ** -0.5) < 1e-15


def test_lists_of_what_is_refused_are_empty():
    """The lists of tiles, items and parts, and the scratch, of sizes that no launch takes: in a process of its own, since a division by zero or a list without an end would be
    this one's."""
    import subprocess
    import sys
    from pathlib import Path
    cases = [("items", a) for a in ((0, 300, 2, 8, 0), (1, 0, 2, 8, 0), (1, 300, 0, 8, 0), (1, 300, 2, 0, 0), (1, 300, 2, 8, -1), (1, 300, 2, 8, 8), (60000, 60000, 2, 8, 0))]
    cases += [(c, a) for c in ("blocks", "keys") for a in ((0, 4, 1, 0), (300, 0, 1, 0), (300, 4, -1, 0), (300, 4, 1, 3), (300, 4, 1, -1))]
    for sizes in ((0, 300, 2, 1, 4, 1), (1, 0, 2, 1, 4, 1), (1, 300, 2, 0, 4, 1), (1, 300, 1, 2, 4, 1), (1, 300, 3, 2, 4, 1), (1, 300, 2, 1, 0, 1), (1, 300, 2, 1, 4, -1),
                  (60000, 60000, 2, 1, 4, 1)):
        cases += [("walk", sizes + (148,)), ("bwd_scratch", sizes)]
    cases.append(("walk", (1, 300, 2, 1, 4, 1, 0)))
    code = "from cai_b200.ops import lib\n"
    for name, args in cases:
        args = ", ".join(map(str, args + (() if name == "bwd_scratch" else (None, 0))))
        code += f"got = lib().cai_flash_attn_window_{name}({args}); assert got == 0, ('{name}', {args}, got)\n"
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])


@pytest.mark.parametrize("change", [dict(B=65536, S=1), dict(nh=65536, ld=65538 * 128, ldq=65538 * 128), dict(B=32768, S=32768, nh=2)], ids=str)
def test_refusals_of_sizes_say_the_limits(change):
    """The limits as the docstring has them."""
    from cai_b200 import ops
    assert "65535 sequences" in ops.flash_attn_window_fwd.__doc__ and "65535 heads" in ops.flash_attn_window_fwd.__doc__
    for name in ("fwd", "bwd"):
        with pytest.raises(ops.KernelError, match="65535 sequences, 65535 heads and fewer than 2\\^30 rows"):
            ops.check(getattr(ops.calls(), f"cai_flash_attn_window_{name}")(*_window(name, **change)), "flash_attn_window")
