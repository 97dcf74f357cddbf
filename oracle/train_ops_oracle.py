"""Oracle of the training and position-dependent operators (star_layer_norm_train / _bwd, star_pos_attn_fwd / _bwd): the formulas in 64-bit
torch on the CPU, and for each output how far a kernel may be off that holds sums in fp32 and rounds what include/star_hip.h says it
rounds, each rounding by half a step of the type (`u`) relative to the value."""
import math

import torch

F = torch.float64
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------------- LayerNorm
def layer_norm_forward(x, gamma, beta, eps):
    x = x.to(F)
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    g = gamma.to(F) if gamma is not None else torch.ones(x.shape[1], dtype=F)
    b = beta.to(F) if beta is not None else torch.zeros(x.shape[1], dtype=F)
    return xh * g + b, torch.cat([mean, rstd], 1)


def layer_norm_backward(dy, x, gamma, eps):
    x, dy = x.to(F), dy.to(F)
    n = x.shape[1]
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    a = dy * gamma.to(F) if gamma is not None else dy
    dx = rstd * (a - a.sum(1, keepdim=True) / n - xh * (a * xh).sum(1, keepdim=True) / n)
    return dx, (dy * xh).sum(0), dy.sum(0)


# ------------------------------------------------------------------------------------------------------------- attention
def visible(Nq, Nk, left=-1, right=-1, sinks=0, start=None, n=None):
    p = (Nk - Nq if start is None else int(start)) + torch.arange(Nq)[:, None]
    j = torch.arange(Nk)[None, :]
    n = Nk if n is None else max(0, min(Nk, int(n)))
    ok = (j < n).expand(Nq, Nk).clone()
    if right >= 0:
        ok &= j <= p + right
    if left >= 0:
        ok &= (j >= p - left) | (j < sinks)
    return ok, j - p


def bucket_scheme(num_buckets, distance, bidirectional):
    out = []
    for rel in range(-distance, distance + 1):
        n = num_buckets // 2 if bidirectional else num_buckets
        first = n if bidirectional and rel > 0 else 0
        d = abs(rel) if bidirectional else max(0, -rel)
        near = n // 2
        if d < near:
            out.append(first + d)
            continue
        k = 0
        while near and k + 1 < n - near and d ** (n - near) * near ** (k + 1) >= near ** (n - near) * distance ** (k + 1):
            k += 1
        out.append(first + near + k)
    return out


def pos_attention(q, k, v, heads, kv_heads, scale, left=-1, right=-1, sinks=0, q_start=None, kv_len=None, bias=None, dout=None, tight=False):
    """q [B, Nq, heads*64], k, v [B or 1, Nk, kv_heads*64] (any float type) -> dict of 64-bit out, lse and, with dout, dq, dk, dv, dtable;
    `tol_*` beside each: the elementwise bound for the inputs' type.
    tight: f16's absolute half step for dS by rows and key blocks.  A kernel rounds 2^e dS with max|dP| 2^e >= 2^13, the maximum over what the row
    sees (dq) or over the rows of the 64-row tiles that see some of the 128 keys of a block (dk): a half step is then 2^-25 2^-13 max|dP|."""
    T = q.dtype
    u = half_step(T)
    sub = 2.0 ** -25 if T == torch.float16 else 0.0          # f16's absolute half step below its normal range
    B, Nq, _ = q.shape
    Nk, S, G = k.shape[1], k.shape[0], heads // kv_heads
    Q, K, V = (t.to(F).reshape(t.shape[0], t.shape[1], -1, 64) for t in (q, k, v))
    r = {n: torch.zeros(B, Nq, heads, 64, dtype=F) for n in ("out", "tol_out")}
    r["lse"], r["tol_lse"] = (torch.full((B, heads, Nq), -math.inf, dtype=F), torch.zeros(B, heads, Nq, dtype=F))
    if dout is not None:
        DO = dout.to(F).reshape(B, Nq, heads, 64)
        for n in ("dq", "tol_dq"):
            r[n] = torch.zeros(B, Nq, heads, 64, dtype=F)
        for n in ("dk", "tol_dk", "dv", "tol_dv"):
            r[n] = torch.zeros(S, Nk, kv_heads, 64, dtype=F)
        if bias is not None:
            r["dtable"], r["tol_dtable"] = torch.zeros(bias[0].shape, dtype=F), torch.zeros(bias[0].shape, dtype=F)
        biggest = float(DO.abs().max()) if DO.numel() else 0.0
    step, oks = torch.zeros(B, heads, Nq, dtype=F), []
    for b in range(B):
        ok, rel = visible(Nq, Nk, left, right, sinks, None if q_start is None else q_start[b], None if kv_len is None else kv_len[b])
        oks.append(ok)
        seen = ok.any(1, keepdim=True)
        if bias is not None:
            R = (len(bias[1]) - 1) // 2
            which = torch.as_tensor(bias[1])[rel.clamp(-R, R) + R]
        for h in range(heads):
            qh, kh, vh = Q[b, :, h], K[b % S, :, h // G], V[b % S, :, h // G]
            kh, vh = (torch.where(ok.any(0)[:, None], t, torch.zeros_like(t)) for t in (kh, vh))    # what no row sees is not there
            s = scale * (qh @ kh.T)
            mag = abs(scale) * (qh.abs() @ kh.abs().T)
            if bias is not None:
                s = s + bias[0].to(F)[:, h][which]
            s = torch.where(ok, s, torch.full_like(s, -math.inf))
            m = torch.where(seen, s.amax(1, keepdim=True) if Nk else torch.zeros(Nq, 1, dtype=F), torch.zeros(Nq, 1, dtype=F))
            m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
            e = torch.exp(s - m)
            l = e.sum(1, keepdim=True)
            P = e / torch.where(l > 0, l, torch.ones_like(l))
            # fp32: a score is a sum of 64 products (64 roundings of its magnitude), scaled, biased and exponentiated (a few more of its size)
            sf = torch.where(torch.isfinite(s), s.abs(), torch.zeros_like(s))
            es = ((70 * mag + 8 * sf) * U32).amax(1, keepdim=True) if Nk else torch.zeros(Nq, 1, dtype=F)
            ep = 2 * es + (16 + Nk / 8) * U32                # of P: numerator and denominator, the denominator's chain of adds
            o = P @ vh
            r["out"][b, :, h] = o
            r["tol_out"][b, :, h] = u * o.abs() + (u * (1 + u) + ep) * (P @ vh.abs()) + sub * vh.abs().sum(0) + sub + 1e-30
            r["lse"][b, h] = torch.where(l > 0, m + torch.log(l), torch.full_like(l, -math.inf))[:, 0]
            r["tol_lse"][b, h] = (es + (16 + Nk / 8) * U32 + 4 * U32 * r["lse"][b, h].abs().nan_to_num(posinf=0)[:, None])[:, 0]
            if dout is None:
                continue
            g = DO[b, :, h]
            dp = g @ vh.T
            dpm = g.abs() @ vh.abs().T
            delta = (P * dp).sum(1, keepdim=True)
            dS = P * (dp - delta)
            # dS: P off by ep (of P and, through it, delta), dP and delta sums of 64 roundings
            dm = (P * dpm).sum(1, keepdim=True)
            sole = (ok.sum(1, keepdim=True) == 1)
            eS = P * ((ep + 70 * U32) * ((dp - delta).abs() + 2 * dm) + 70 * U32 * dpm)
            eS = torch.where(sole, torch.zeros_like(eS), eS)
            rS = u * dS.abs() + eS * (1 + u)
            top = float(g.abs().max()) if g.numel() else 0.0
            r["dq"][b, :, h] = scale * (dS @ kh)
            least = sub * top * kh.abs().sum(0)
            if tight:
                step[b, h] = sub * 2.0 ** -13 * (dp.abs() * ok).amax(1)
                least = step[b, h][:, None] * (ok.to(F) @ kh.abs())
            r["tol_dq"][b, :, h] = u * r["dq"][b, :, h].abs() + abs(scale) * (rS @ kh.abs() + least) + sub + 1e-30
            kvh = h // G
            r["dk"][b % S, :, kvh] += scale * (dS.T @ qh)
            r["tol_dk"][b % S, :, kvh] += abs(scale) * (rS.T @ qh.abs() + (0.0 if tight else sub * biggest * qh.abs().sum(0))) + Nq * U32 * abs(scale) * (dS.abs().T @ qh.abs())
            r["dv"][b % S, :, kvh] += P.T @ g
            r["tol_dv"][b % S, :, kvh] += (u + Nq * U32) * (P.T @ g.abs()) + (ep * P).T @ g.abs() + sub * 2.0 ** -10 * g.abs().sum(0)
            if bias is not None:
                r["dtable"][:, h].index_add_(0, which.flatten(), dS.flatten())
                r["tol_dtable"][:, h].index_add_(0, which.flatten(), (eS + (Nq + Nk) * U32 * dS.abs()).flatten())
    if dout is not None and tight:
        for j in range(0, Nk, 128):
            blk = slice(j, j + 128)
            # the tokens that see some of these keys, and those that may share a tile of 64 rows with them
            near = [torch.nn.functional.max_pool1d(o[:, blk].any(1).to(F)[None, None], 127, 1, 63)[0, 0] for o in oks]
            for b in range(B):
                for kvh in range(kv_heads):
                    same = range(B) if S == 1 else [b]
                    most = max(float((step[c, kvh * G:(kvh + 1) * G] * near[c]).max()) for c in same)
                    for h in range(kvh * G, (kvh + 1) * G):
                        r["tol_dk"][b % S, blk, kvh] += abs(scale) * most * (oks[b][:, blk].to(F).T @ Q[b, :, h].abs())
    if dout is not None:
        for n in ("dk", "dv"):
            r["tol_" + n] += u * r[n].abs() + sub + 1e-30
        if bias is not None:
            r["tol_dtable"] += 1e-30
    for n in list(r):
        if r[n].dim() == 4:
            r[n] = r[n].reshape(r[n].shape[0], r[n].shape[1], -1)
    return r
