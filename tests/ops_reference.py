"""64-bit references of the tensor operators (``ops.py``), written from their definitions, and the
error bounds that the tests hold the kernels to.

u = 2^-24 is half a step of fp32.  A result rounded to type t is off by at most finfo(t).eps / 2 of
its value, which every bound adds at the end; below t's normal range the step is finfo(t).tiny *
eps.  First-order bounds are doubled (``SLACK``) for the terms of second order and for the hardware
exp2 / log2, whose error (1 ulp) is counted as 2 u.
"""
import torch

U = 2.0 ** -24
SLACK = 2.0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(ref, dtype):
    """The most that rounding `ref` to dtype takes off."""
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps / 2) + fi.tiny * fi.eps


def check(got, ref, bound, what=""):
    """Every finite value within its bound; NaN and infinities where the reference has them."""
    got = got.detach().double().cpu()
    ref, bound = ref.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what + ": NaN elsewhere"
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin].nan_to_num(7.0), ref[~fin].nan_to_num(7.0)), what + ": infinities"
    bound = bound.expand(ref.shape)[fin]
    off = (got[fin] - ref[fin]).abs()
    over = off > bound
    if bool(over.any()):
        i = int((off / bound.clamp_min(1e-300)).argmax())
        raise AssertionError(f"{what}: {int(over.sum())} of {over.numel()} outside; the furthest: "
                             f"{float(got[fin][i]):.9g} for {float(ref[fin][i]):.9g}, off "
                             f"{float(off[i]):.3g}, bound {float(bound[i]):.3g}")


# ---- embedding -----------------------------------------------------------------------------------
def embed(weight, ids, scale):
    ok = (ids >= 0) & (ids < weight.shape[0])
    out = weight.double()[ids.clamp(0, weight.shape[0] - 1)] * scale
    out[~ok] = float("nan")
    # the scale is rounded to fp32 and so is the product
    return out, SLACK * 2 * U * out.abs() + rounded(out, weight.dtype)


def embed_grad(dout, ids, V, scale, pad, dtype):
    """(gradient, bound): m terms summed in fp32 in any order are off by (m - 1) u of their
    magnitudes' sum; the scale and the product add 2 u."""
    d = dout.shape[-1]
    ids, dout = ids.reshape(-1).cpu(), dout.reshape(-1, d).double().cpu()
    ok = (ids >= 0) & (ids < V)
    if pad is not None:
        ok &= ids != pad
    ids, dout = ids[ok], dout[ok]
    z = torch.zeros(V, d, dtype=torch.float64, device=dout.device)
    ref = z.index_add(0, ids.long(), dout) * scale
    mag = z.index_add(0, ids.long(), dout.abs()) * abs(scale)
    m = torch.bincount(ids.long(), minlength=V)[:, None]
    return ref, SLACK * (m + 2) * U * mag + rounded(ref, dtype)


# ---- cross attention -----------------------------------------------------------------------------
def attention(q, k, v, keep, scale, dout=None):
    """{"out": (ref, bound), and with dout "dq", "dk", "dv"}.

    Bounds.  A score is off by ds = (D + 3) u scale sum |q||k| + 2 u |s|, so a probability by a factor
    e = 2 max_j ds_j + (Lk + 20) u (its own exponent, the row's maximum, the sum's additions), and
    p^ = p (1 + e).  bf16 rounds p and dS once more: r = 2^-8 each (0 for the others, whose
    products are exact in fp32).
      out: sum_j p |v| (e + r + Lk u)
      dV:  sum_i p |dO| (e + r + R u), R rows
      dS:  x = p ((e + r) |dP - delta| + D u sum |dO||v| + d_delta).  delta is sum |dO O| of an O whose
           weights w add up to 1 whatever their errors, so sum (w - p) dP = sum (w - p) (dP - delta)
           and w - p is at most 2 (e + r) p: d_delta = 2 (e + r) sum p |dP - delta| + (D u + r^2 + u)
           sum |dO O|, O itself being kept to two bf16 (r^2)
      dQ:  scale sum_j (x + p |dP - delta| Lk u) |k|;   dK with R and |q|
    fp32 has no normal number under 2^-126: exp2 of less than -126 may come out 0, and so may a
    product's operand or sum below it, so every p carries 2^-125 besides (two such steps): `least`."""
    least = 2.0 ** -125
    dt = q.dtype
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    r = 2.0 ** -8 if dt == torch.bfloat16 else 0.0
    q_, k_, v_ = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    if keep is not None:
        keep = keep.expand(B, Lk)[:, None, :, None]
        k_ = torch.where(keep, k_, 0.0)
        v_ = torch.where(keep, v_, 0.0)
    kk, vv = k_.repeat_interleave(G, 1), v_.repeat_interleave(G, 1)

    def mm(a, b):
        return torch.matmul(a.contiguous(), b.contiguous())

    def t_(a):
        return a.transpose(-1, -2)
    s = mm(q_, t_(kk)) * scale
    ds = (D + 3) * U * abs(scale) * mm(q_.abs(), t_(kk.abs())) + 2 * U * s.abs()
    live = torch.ones(B, 1, 1, Lk, dtype=torch.bool, device=q.device)
    if keep is not None:
        live = live & t_(keep)
    s = torch.where(live, s, float("-inf"))
    some = live.any(-1, keepdim=True) if Lk else torch.zeros(B, 1, 1, 1, dtype=torch.bool,
                                                             device=q.device)
    if Lk == 0:
        p = s
        e = torch.zeros(B, H, Lq, 1, dtype=torch.float64, device=q.device)
    else:
        p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), -1), 0.0)
        e = 2 * torch.where(live, ds, 0.0).amax(-1, keepdim=True) + (Lk + 20) * U
    out = mm(p, vv)
    b_out = SLACK * (mm(p, vv.abs()) * (e + r + Lk * U) + least * vv.abs().sum(-2, True)) + rounded(
        out, dt)
    res = {"out": (out.transpose(1, 2), b_out.transpose(1, 2))}
    if dout is None:
        return res
    R = G * Lq
    do = dout.detach().double().transpose(1, 2)
    dp = mm(do, t_(vv))
    delta = (do * out).sum(-1, keepdim=True)
    g = torch.where(live & some, p * (dp - delta), 0.0)
    spread = (p * (dp - delta).abs()).sum(-1, keepdim=True)
    d_delta = 2 * (e + r) * spread + (D * U + r * r + U) * (do * out).abs().sum(-1, keepdim=True)
    x = (p * (e + r) + least) * (dp - delta).abs() + p * (
        D * U * mm(do.abs(), t_(vv.abs())) + d_delta)
    dq = scale * mm(g, kk)
    b_dq = SLACK * abs(scale) * mm(x + g.abs() * Lk * U, kk.abs())

    def heads(a):  # a key head's gradient sums its query heads'
        return a.reshape(B, Hkv, G, Lk, D).sum(2)
    dk = scale * heads(mm(t_(g), q_))
    b_dk = SLACK * abs(scale) * heads(mm(t_(x + g.abs() * R * U), q_.abs()))
    dv = heads(mm(t_(p), do))
    b_dv = SLACK * heads(mm(t_(p * (e + r + R * U) + least), do.abs()))
    for name, ref, bound in (("dq", dq, b_dq), ("dk", dk, b_dk), ("dv", dv, b_dv)):
        res[name] = (ref.transpose(1, 2), (bound + rounded(ref, dt)).transpose(1, 2))
    return res


# ---- preference ----------------------------------------------------------------------------------
def preference(logits, labels, ref_logps=None, beta=0.1, smooth=0.0, upstream=1.0, dlogps=None):
    """{"logps", "loss", "dlogits"}: (ref, bound) each.

    Bounds.  exp(x - m) in fp32 is off by (|x - m| + 3) 2 u of itself; the sum by that, weighted, and
    (V / 256 + 40) u for its additions (256 threads, each a chain); a position's log-probability by
    that and 2 u (|x_y - m| + |log sum| + 1), a sequence's by the sum and its own rounding.  A margin
    is off by beta times its two answers' errors, the loss by as much (its slope is at most 1), and
    dlp by beta / P times a quarter of it."""
    x = logits.detach().double()
    S, T, V = x.shape
    ok = (labels >= 0) & (labels < V)
    valid = labels >= 0
    m = x.amax(-1, keepdim=True)
    ex = (x - m).exp()
    z = ex.sum(-1, keepdim=True)
    p = ex / z
    e_exp = ((x - m).abs().nan_to_num(0.0, 0.0, 0.0) + 3) * 2 * U
    e_sum = (p * e_exp).sum(-1, keepdim=True) + (V / 256 + 40) * U
    at = labels.clamp(0, V - 1).long()[..., None]
    xy = x.gather(-1, at)
    tok = (xy - m - z.log())[..., 0]
    tok = torch.where(ok, tok, float("nan"))
    tok = torch.where(valid, tok, 0.0)
    b_tok = (e_sum + 2 * U * ((xy - m).abs() + z.log().abs() + 1))[..., 0]
    b_tok = torch.where(valid, b_tok, 0.0)  # an ignored row's logit may be infinite
    logps = tok.sum(-1)
    b_lp = SLACK * b_tok.sum(-1) + U * logps.abs() + 1e-30
    res = {"logps": (logps, b_lp)}
    if ref_logps is not None:
        P = S // 2
        rf = ref_logps.double()
        mg = beta * ((logps[:P] - logps[P:]) - (rf[:P] - rf[P:]))
        b_mg = abs(beta) * SLACK * (b_tok.sum(-1)[:P] + b_tok.sum(-1)[P:]) + 4 * U * mg.abs()
        sp = torch.nn.functional.softplus
        loss = ((1 - smooth) * sp(-mg) + smooth * sp(mg)).mean()
        res["loss"] = (loss, b_mg.mean() + 2 * U * loss.abs() + 1e-30)
        g = beta / P * (smooth - torch.sigmoid(-mg))
        b_g = abs(beta) / P * b_mg / 4 + 4 * U * g.abs()
        dlogps, b_d = torch.cat([g, -g]), torch.cat([b_g, b_g])
    elif dlogps is not None:
        dlogps = dlogps.double()
        b_d = torch.zeros_like(dlogps)
    else:
        return res
    c, b_c = (dlogps * upstream)[:, None, None], (b_d * abs(upstream))[:, None, None]
    hot = torch.zeros_like(x).scatter_(-1, at, 1.0)
    dx = torch.where(valid[..., None], c * (hot - p), 0.0)
    dx = torch.where((valid & ~ok)[..., None], float("nan"), dx)
    b = c.abs() * p * SLACK * (e_exp + e_sum + 4 * U) + SLACK * (b_c + 2 * U * c.abs()) * (
        hot - p).abs() + U * c.abs() * hot
    res["dlogits"] = (dx, torch.where(valid[..., None], b, 0.0).nan_to_num(0.0) + rounded(
        dx.nan_to_num(0.0), logits.dtype))
    return res
