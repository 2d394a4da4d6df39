"""What the operators of a layer's attention half are measured on: windowed attention with sinks, rotary positions of several axes, and
RMSNorm that adds the residual and leaves its rows in e4m3.

  norm     ``h = x + residual``, its RMSNorm in e4m3 with a scale for each row and 128 columns, as the block-scaled product reads it; where a
           weight gradient will need it, the bf16 rows too.
  rope     the q and k heads of a packed activation turned in place by the positions of several axes (time, height, width);
           with ``inverse``, back, as a backward pass does.
  window   causal grouped-query attention in which a token sees the ``window`` tokens up to itself and the first ``sinks``; with
           ``train``, the gradients of q, k and v as well.

A case is a dict of plain values. ``prepare`` makes its inputs, ``run`` one pass: in elementary torch operations, or, where ``own`` is true,
through ``cai_b200.ops``. ``exact`` gives the same from the definitions in 64 bits.
"""
import math

import torch

own = False          # whether run() calls the framework's operators

HD = 128             # the head dimension of the framework's attention
THETA = 10000.0
EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # the smallest layers: the widths of configs/tiny.cfg on its batch of two sequences of 128 tokens; launches count, not bytes
        dict(kind="norm", name="norm_tiny", rows=256, hidden=256, residual=1, keep_y=1),
        # an evaluation pass over an odd number of tokens: the product before has added the residual, no gradient will be asked for
        dict(kind="norm", name="norm_odd", rows=1777, hidden=1408, residual=0, keep_y=0),
        # a training batch at the width of the 8B-class model (configs/b200_fsdp8b.cfg)
        dict(kind="norm", name="norm_wide", rows=16384, hidden=4096, residual=1, keep_y=1),
        # one image's tokens in the smallest model
        dict(kind="rope", name="rope_tiny", tokens=256, heads=2, kv_heads=1, sections="22,21,21", interleaved=0, inverse=0, span=64),
        # odd number of tokens and heads that divide nothing; the backward pass's turn
        dict(kind="rope", name="rope_odd", tokens=5003, heads=9, kv_heads=3, sections="16,24,24", interleaved=0, inverse=1, span=4000),
        # a long video at the 8B-class model's heads, frames far into it, axes spread over all frequencies
        dict(kind="rope", name="rope_long", tokens=32768, heads=32, kv_heads=8, sections="24,20,20", interleaved=1, inverse=0, span=200000),
        # a training step of the smallest model: two short sequences
        dict(kind="window", name="window_tiny", train=1, batch=2, seq=128, heads=2, kv_heads=1, window=64, sinks=4),
        # short sequences of odd length, no sinks, forward alone
        dict(kind="window", name="window_odd", train=0, batch=3, seq=1000, heads=9, kv_heads=3, window=200, sinks=0),
        # evaluation of a long text at the benchmark model's heads (configs/b200_tp8.cfg), a wide window
        dict(kind="window", name="window_wide", train=0, batch=1, seq=16384, heads=16, kv_heads=8, window=4096, sinks=4),
        # fine-tuning on one short document: one kv head, odd length, a window that is longer than the sequence
        dict(kind="window", name="window_few_rows", train=1, batch=1, seq=333, heads=8, kv_heads=1, window=512, sinks=1),
        # a training batch of the benchmark model
        dict(kind="window", name="window_train", train=1, batch=4, seq=4096, heads=16, kv_heads=8, window=1024, sinks=4),
        # one GPU's heads of a sharded model on a very long sequence, sinks that fill more than a tile
        dict(kind="window", name="window_train_long", train=1, batch=1, seq=32768, heads=4, kv_heads=1, window=2048, sinks=130),
    ]


# ---------------------------------------------------------------------------- more cases of the same ranges
MOST_NORM = 16384 * 4096             # elements of a norm
MOST_ROPE = 32768 * 40               # heads of all tokens that are turned
MOST_SCORES = 1 << 32                # batch x heads x seq x seq: what the plain form holds of scores
MOST_PAIRS = {0: 16 * 16384 * 4096, 1: 64 * 4096 * 1024}     # visible (query, key) pairs: forward alone, with the gradients


def _log(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / multiple)) * multiple))


def draw(rng):
    while True:
        kind = rng.choices(["norm", "rope", "window"], [2, 2, 4])[0]
        if kind == "norm":
            c = dict(kind=kind, rows=_log(rng, 1, 32768), hidden=_log(rng, 128, 8192, 128), residual=int(rng.random() < 0.6), keep_y=int(rng.random() < 0.6))
            if c["rows"] * c["hidden"] > MOST_NORM:
                continue
        elif kind == "rope":
            kv = rng.choice([1, 2, 3, 4, 8])
            c = dict(kind=kind, tokens=_log(rng, 1, 32768), heads=kv * rng.choice([1, 2, 3, 4]), kv_heads=kv,
                     sections=rng.choice(["64", "32,32", "16,24,24", "24,20,20", "22,21,21", "16,16,16,16"]), interleaved=int(rng.random() < 0.4),
                     inverse=int(rng.random() < 0.4), span=_log(rng, 1, 1 << 20))
            if c["tokens"] * (c["heads"] + kv) > MOST_ROPE or [_axis_of_pairs(c).count(a) for a in range(len(_sections(c)))] != _sections(c):
                continue
        else:
            kv = rng.choice([1, 2, 3, 4, 8])
            c = dict(kind=kind, train=int(rng.random() < 0.6), batch=_log(rng, 1, 16), seq=_log(rng, 1, 32768), heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv,
                     window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, rng.randint(1, 64), _log(rng, 64, 512)]))
            if c["batch"] * c["heads"] * c["seq"] ** 2 > MOST_SCORES or c["batch"] * c["heads"] * _pairs(c) > MOST_PAIRS[c["train"]]:
                continue
        return c


def _pairs(case):
    """How many (query, key) pairs of one head are visible."""
    S, W, n = case["seq"], case["window"], case["sinks"]
    w = min(W, S)
    total = w * (w + 1) // 2 + (S - w) * w
    far = S - w                       # queries whose window has left the first tokens behind: query w + i no longer reaches keys 0 .. i
    m = min(n, far)
    return total + m * (m + 1) // 2 + (far - m) * n if far else total


# ---------------------------------------------------------------------------- inputs
def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def _axis_of_pairs(case):
    """The axis whose position turns pair i of a head, for each i: one run of pairs after the other, or, interleaved, pair i belongs to axis
    i mod the number of axes as long as that axis has pairs left, and to the first after that (which has to come out at its number)."""
    sections = _sections(case)
    if not case["interleaved"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    m = len(sections)
    return [i % m if i // m < sections[i % m] else 0 for i in range(HD // 2)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(torch.bfloat16)

    if case["kind"] == "norm":
        rows, H = case["rows"], case["hidden"]
        # a residual stream whose channels differ in size, a few of them much larger than the rest, and a branch's output to be added
        channel = torch.exp(0.7 * torch.randn(H, device="cuda", generator=g))
        x = (torch.randn(rows, H, device="cuda", generator=g) * channel).to(torch.bfloat16)
        return dict(case=case, x=x, residual=normal(rows, H, scale=0.5) if case["residual"] else None,
                    gain=(1.0 + 0.2 * torch.randn(H, device="cuda", generator=g)).to(torch.bfloat16))
    if case["kind"] == "rope":
        T, nh, nkv = case["tokens"], case["heads"], case["kv_heads"]
        axes = len(_sections(case))
        # the first axis runs on far into the sequence, the others stay inside a picture
        pos = torch.randint(0, max(1, case["span"]), (axes, T), device="cuda", generator=g, dtype=torch.int32)
        pos[1:] %= 128
        state = dict(case=case, qkv=normal(T, (nh + 2 * nkv) * HD), pos=pos, sections=_sections(case))
        # what a program keeps with its model: radians a position, pair by pair
        state["freqs"] = THETA ** (-torch.arange(HD // 2, device="cuda", dtype=torch.float64) / (HD // 2))
        state["axis"] = torch.tensor(_axis_of_pairs(case), device="cuda")
        return state
    B, S, nh, nkv = case["batch"], case["seq"], case["heads"], case["kv_heads"]
    state = dict(case=case, qkv=normal(B * S, (nh + 2 * nkv) * HD))
    if case["train"]:
        state["dout"] = normal(B * S, nh * HD)
    return state


# ---------------------------------------------------------------------------- one pass
def run(state):
    return {"norm": _norm, "rope": _rope, "window": _window}[state["case"]["kind"]](state)


def _norm(state):
    case = state["case"]
    if own:
        from cai_b200 import ops
        h, q, s, rstd, y = ops.add_rmsnorm_quant(state["x"], state["residual"], state["gain"], EPS, keep_y=bool(case["keep_y"]))
    else:
        rows, H = state["x"].shape
        h = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).to(torch.bfloat16)
        hf = h.float()
        rstd = 1.0 / torch.sqrt((hf * hf).mean(1) + EPS)
        yf = hf * rstd[:, None] * state["gain"].float()
        blocks = yf.view(rows, H // 128, 128)
        s = blocks.abs().amax(2) / E4M3_MAX
        s = torch.where(s > 0, s, torch.ones_like(s))
        q = (blocks / s[:, :, None]).to(torch.float8_e4m3fn).view(rows, H)
        y = yf.to(torch.bfloat16) if case["keep_y"] else None
    return dict(h=h if case["residual"] else None, q=q, s=s, rstd=rstd, y=y)


def _rope(state):
    case, qkv = state["case"], state["qkv"]
    nh, nkv = case["heads"], case["kv_heads"]
    if own:
        from cai_b200 import ops
        return ops.rope_apply_axes_(qkv, state["freqs"], state["pos"], nh, nkv, HD, state["sections"], interleaved=bool(case["interleaved"]),
                                    inverse=bool(case["inverse"]))
    # far positions: the angles in 64 bits
    angle = state["pos"][state["axis"]].t().double() * state["freqs"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["inverse"]:
        sin = -sin
    x = qkv.view(qkv.shape[0], nh + 2 * nkv, HD)[:, :nh + nkv]
    a, b = x[..., :HD // 2].float(), x[..., HD // 2:].float()
    x[..., :HD // 2] = a * cos - b * sin
    x[..., HD // 2:] = b * cos + a * sin
    return qkv


def _window(state):
    case, qkv = state["case"], state["qkv"]
    B, S, nh, nkv, W, sinks = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "window", "sinks"))
    if own:
        from cai_b200 import ops
        out, lse = ops.flash_attn_window_fwd(qkv, B, S, nh, nkv, HD, W, sinks)
        if not case["train"]:
            return dict(out=out, lse=lse)
        return dict(out=out, lse=lse, dqkv=ops.flash_attn_window_bwd(qkv, out, state["dout"], lse, B, S, nh, nkv, HD, W, sinks))
    rep, scale = nh // nkv, HD ** -0.5
    x = qkv.float().view(B, S, nh + 2 * nkv, HD).transpose(1, 2)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv].repeat_interleave(rep, 1), x[:, nh + nkv:].repeat_interleave(rep, 1)
    i, j = torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None]
    hidden = (j > i) | ((j <= i - W) & (j >= sinks))
    p = (q @ k.transpose(2, 3)).mul_(scale).masked_fill_(hidden, -math.inf)
    m = p.amax(3, keepdim=True)
    p = p.sub_(m).exp_()
    l = p.sum(3, keepdim=True)
    p = p.div_(l)
    o = p @ v
    got = dict(out=o.transpose(1, 2).reshape(B * S, nh * HD).to(torch.bfloat16), lse=(m + l.log())[..., 0])
    if case["train"]:
        do = state["dout"].float().view(B, S, nh, HD).transpose(1, 2)
        dv = p.transpose(2, 3) @ do
        ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(scale)
        dq, dk = ds @ k, ds.transpose(2, 3) @ q
        # a kv head's gradient is the sum over its query heads
        dk, dv = (t.reshape(B, nkv, rep, S, HD).sum(2) for t in (dk, dv))
        got["dqkv"] = torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(B * S, -1).to(torch.bfloat16)
    return got


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "norm":
        rows, H = case["rows"], case["hidden"]
        n = rows * H
        bytes_ = n * (2 + 4 * case["residual"] + 2 * case["keep_y"] + 1) + rows * (H // 128 * 4 + 4) + 2 * H
        return {"bytes": bytes_, "flops": 6 * n}
    if case["kind"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * HD
        return {"bytes": 4 * n + 4 * case["tokens"] * len(_sections(case)), "flops": 3 * n}
    B, S, nh, nkv = case["batch"], case["seq"], case["heads"], case["kv_heads"]
    pairs, tokens = B * nh * _pairs(case), B * S
    qkv, out, lse = tokens * (nh + 2 * nkv) * HD * 2, tokens * nh * HD * 2, tokens * nh * 4
    if not case["train"]:
        return {"bytes": qkv + out + lse, "flops": 4 * HD * pairs}          # scores, and what they weigh
    # with the gradients: the scores again (which need not be kept), dP, dV, dQ, dK; q, k, v once more, dO in, their gradients out
    return {"bytes": 3 * qkv + 3 * out + 2 * lse, "flops": (4 + 10) * HD * pairs}


# ---------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        h = state["x"].double()
        if case["residual"]:
            # the stream is held in bf16: the norm is that of the rounded sum
            h = (h + state["residual"].double()).to(torch.bfloat16).double()
        rstd = (h.square().mean(1) + EPS).rsqrt()
        y = torch.einsum("rc,r,c->rc", h, rstd, state["gain"].double())
        s = y.unflatten(1, (-1, 128)).abs().amax(-1) / E4M3_MAX
        s = s.masked_fill(s == 0, 1.0)
        q = _to_e4m3(y / s.repeat_interleave(128, 1))
        return dict(h=h if case["residual"] else None, q=q, s=s, rstd=rstd, y=y if case["keep_y"] else None)
    if case["kind"] == "rope":
        T, heads = case["tokens"], case["heads"] + case["kv_heads"]
        x = state["qkv"].double().unflatten(1, (-1, 2, HD // 2))
        turned = x[:, :heads]
        angle = torch.empty(T, HD // 2, device="cuda", dtype=torch.float64)
        for i, axis in enumerate(_axis_of_pairs(case)):
            angle[:, i] = state["pos"][axis].double() * math.exp(-i / (HD // 2) * math.log(THETA))
        if case["inverse"]:
            angle = -angle
        z = torch.complex(turned[:, :, 0], turned[:, :, 1]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        x[:, :heads] = torch.stack([z.real, z.imag], 2)
        return x.flatten(1)
    B, S, nh, nkv, W, sinks = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "window", "sinks"))
    rep, scale = nh // nkv, 1.0 / math.sqrt(HD)
    x = state["qkv"].double().view(B, S, nh + 2 * nkv, HD).permute(0, 2, 1, 3)
    out = torch.zeros(B, nh, S, HD, device="cuda", dtype=torch.float64)
    lse = torch.zeros(B, nh, S, device="cuda", dtype=torch.float64)
    dx = torch.zeros_like(x) if case["train"] else None
    step = 512
    for b in range(B):
        q, k, v = x[b, :nh].view(nkv, rep, S, HD), x[b, nh:nh + nkv], x[b, nh + nkv:]
        for q0 in range(0, S, step):
            q1 = min(S, q0 + step)
            # only the keys that some query of the block sees: the first ones, and its windows
            w0 = max(0, q0 - W + 1)
            keys = torch.cat([torch.arange(min(sinks, w0), device="cuda"), torch.arange(w0, q1, device="cuda")])
            i = torch.arange(q0, q1, device="cuda")[:, None]
            seen = (keys <= i) & ((keys > i - W) | (keys < sinks))
            kb, vb, qb = k[:, keys], v[:, keys], q[:, :, q0:q1]
            s = torch.einsum("grqd,gkd->grqk", qb, kb) * scale
            s = torch.where(seen, s, -math.inf)
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - z[..., None])
            o = torch.einsum("grqk,gkd->grqd", p, vb)
            out[b, :, q0:q1] = o.reshape(nh, q1 - q0, HD)
            lse[b, :, q0:q1] = z.reshape(nh, q1 - q0)
            if case["train"]:
                do = state["dout"].double().view(B, S, nkv, rep, HD)[b, q0:q1].permute(1, 2, 0, 3)
                dp = torch.einsum("grqd,gkd->grqk", do, vb)
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dx[b, :nh, q0:q1] = torch.einsum("grqk,gkd->grqd", ds, kb).reshape(nh, q1 - q0, HD)
                dx[b, nh:nh + nkv].index_add_(1, keys, torch.einsum("grqk,grqd->gkd", ds, qb))
                dx[b, nh + nkv:].index_add_(1, keys, torch.einsum("grqk,grqd->gkd", p, do))
    got = dict(out=out.permute(0, 2, 1, 3).reshape(B * S, nh * HD), lse=lse)
    if case["train"]:
        got["dqkv"] = dx.permute(0, 2, 1, 3).reshape(B * S, -1)
    return got


def _to_e4m3(x):
    """The nearest number with three bits behind the leading one, the smallest exponent -6, at most 448; ties go to the even one."""
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
