"""The cases on which the training and serving operators of star_amd are measured.

Three operators, each in every direction that a program calls:

* LayerNorm with saved row statistics, and its backward pass with the reduction of the weight's gradient
  (`Context.layer_norm_train`, `Context.layer_norm_backward`);
* attention with a learned relative position bias by buckets, its backward pass with the table's gradient, and its single-token form
  (`Context.pos_attention`, `Context.pos_attention_backward`, `Context.rel_buckets`);
* attention with a sliding window and a few first tokens that stay visible, as a whole sequence, as a chunk against a cache, as a single
  token against a cache, and its backward pass (the same entry points with `window` and `sinks`).

`own` false: elementary torch operations in 32 bits.  `own` true: the framework's entry points.
"""
import math

import torch

own = False

D = 64                      # head width of every attention layer of this repository
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases
def _norm(name, kind, dtype, rows, C, affine=True):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "C": C, "affine": affine}


def _attn(name, kind, dtype, B, Nq, Nk, H, KH, left=-1, right=-1, sinks=0, buckets=0, distance=0, both=True, ragged=0.0, cache=False, scale=0.125, lse=False):
    return {"name": name, "kind": kind, "dtype": dtype, "B": B, "Nq": Nq, "Nk": Nk, "H": H, "KH": KH, "left": left, "right": right, "sinks": sinks,
            "buckets": buckets, "distance": distance, "both": both, "ragged": ragged, "cache": cache, "scale": scale, "lse": lse}


def listed():
    return [
        # two prompts (a guided pair) through a LayerNorm of the text tower: the smallest call, all latency
        _norm("norm_fwd_prompts", "norm_fwd", "f16", 2 * 77, 1024),
        # every token of a 32-frame clip at the first level of the denoiser: all bandwidth
        _norm("norm_fwd_clip", "norm_fwd", "f16", 32 * 122 * 216, 320),
        # a fine-tuning step of the text tower on eight prompts: the reduction over rows is short, the launches count
        _norm("norm_bwd_prompts", "norm_bwd", "bf16", 8 * 77, 1024),
        # a fine-tuning step of the denoiser's second level on a 32-frame clip
        _norm("norm_bwd_clip", "norm_bwd", "f16", 32 * 62 * 108, 640),
        # a batch of padded prompts of up to 226 tokens through a text encoder layer with bucketed bias (scale 1: such encoders do not scale),
        # with the row statistics that its backward pass takes
        _attn("relpos_fwd_prompts", "attn_fwd", "f16", 8, 226, 226, 32, 32, buckets=32, distance=128, ragged=0.8, scale=1.0, lse=True),
        # the same layer trained
        _attn("relpos_bwd_prompts", "attn_bwd", "bf16", 4, 226, 226, 16, 16, buckets=32, distance=128, ragged=0.8, scale=1.0),
        # training on long captions: nearly every tile is past the bias's range, the products count
        _attn("relpos_bwd_long", "attn_bwd", "bf16", 2, 4099, 4099, 16, 16, buckets=32, distance=128, ragged=0.1),
        # a decoder with bucketed bias that writes the next token of sixteen sequences of different lengths
        _attn("relpos_step", "attn_fwd", "bf16", 16, 1, 8200, 16, 16, right=0, buckets=32, distance=128, both=False, ragged=0.7, cache=True),
        # the video transformer's sequence (226 text tokens that every token sees, 13 frames of 30 x 45 tokens), each token seeing four frames either way
        _attn("window_fwd_video", "attn_fwd", "f16", 1, 226 + 13 * 1350, 226 + 13 * 1350, 16, 16, left=4 * 1350, right=4 * 1350, sinks=226),
        # streaming: one new frame of 1350 tokens against a cache of earlier frames, eight frames back, grouped heads
        _attn("window_fwd_chunk", "attn_fwd", "bf16", 1, 1350, 226 + 20 * 1350, 16, 4, left=8 * 1350, right=0, sinks=226, cache=True),
        # the next token of 32 sequences in long caches: only the window and the first tokens are read
        _attn("window_step", "attn_fwd", "bf16", 32, 1, 32800, 32, 8, left=4095, right=0, sinks=64, ragged=0.9, cache=True),
        # training with the window, causal, grouped heads
        _attn("window_bwd", "attn_bwd", "f16", 1, 4500, 4500, 16, 4, left=1023, right=0, sinks=77),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    dtype = rng.choice(["f16", "bf16"])
    what = rng.choice(["norm_fwd", "norm_bwd", "relpos_fwd", "relpos_bwd", "relpos_step", "window_fwd", "window_bwd", "window_chunk", "window_step"])
    if what.startswith("norm"):
        C = _log(rng, 8, 5120)
        if rng.random() < 0.7:
            C = 8 * max(1, C // 8)
        return _norm("", what, dtype, _log(rng, 1, 32 * 122 * 216), C, rng.random() < 0.8)
    KH = rng.choice([1, 2, 4, 5, 8])
    H = KH * rng.choice([1, 1, 2, 4])
    B = _log(rng, 1, 8)
    scale = rng.choice([0.125, 0.125, 1.0])
    bias = {"buckets": rng.choice([8, 32, 32, 64]), "distance": rng.choice([64, 128, 128, 500])}
    band = {"left": _log(rng, 1, 6000), "sinks": rng.choice([0, 1, 4, 77, 226])}
    if what in ("relpos_fwd", "relpos_bwd"):
        N = _log(rng, 1, 4200)
        both = rng.random() < 0.7
        return _attn("", "attn_fwd" if what == "relpos_fwd" else "attn_bwd", dtype, B, N, N, H, KH, right=-1 if both else 0, both=both,
                     ragged=rng.choice([0.0, 0.5, 1.0]), scale=scale, lse=what == "relpos_fwd", **bias)
    if what == "relpos_step":
        return _attn("", "attn_fwd", dtype, _log(rng, 1, 32), 1, _log(rng, 1, 9000), H, KH, right=0, both=False, ragged=rng.choice([0.0, 0.7, 1.0]),
                     cache=True, scale=scale, **bias)
    if what in ("window_fwd", "window_bwd"):
        N = _log(rng, 1, 9000 if what == "window_fwd" else 4500)
        band["right"] = rng.choice([0, 0, band["left"]])
        return _attn("", "attn_fwd" if what == "window_fwd" else "attn_bwd", dtype, min(B, 4), N, N, H, KH, ragged=rng.choice([0.0, 0.5]),
                     lse=what == "window_fwd" and rng.random() < 0.5, **band)
    if what == "window_chunk":
        Nq = _log(rng, 2, 1350)
        return _attn("", "attn_fwd", dtype, min(B, 4), Nq, Nq + _log(rng, 1, 30000), H, KH, right=0, ragged=rng.choice([0.0, 0.5]), cache=True, **band)
    return _attn("", "attn_fwd", dtype, _log(rng, 1, 32), 1, _log(rng, 1, 33000), H, KH, right=0, ragged=rng.choice([0.0, 0.9, 1.0]), cache=True, **band)


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for k in w:
            most[c["kind"], k] = max(most.get((c["kind"], k), 0), w[k])
    while True:
        c = _draw(rng)
        del c["name"]
        if all(v <= most[c["kind"], k] for k, v in work(c).items()) and c.get("B", 1) * c.get("KH", 1) * c.get("Nk", 1) <= 32 * 8 * 32800 and \
                c.get("B", 1) * c.get("H", 1) * c.get("Nq", 1) * c.get("Nk", 1) <= 16 * 17776 ** 2:
            return c


def lengths(c):
    """keys in hand per sequence, and the position of each sequence's first query row"""
    B, Nk, Nq = c["B"], c["Nk"], c["Nq"]
    least = min(Nq, Nk) if c["cache"] else 1
    lens = [max(least, Nk - int(round(c["ragged"] * Nk * b / max(1, B - 1)))) for b in range(B)]
    return lens, [n - Nq if c["cache"] else 0 for n in lens]


def _span(c, n, pos):
    """[lo, hi) of the window of the query at `pos` in a sequence of n keys, and the count of first tokens visible beside it"""
    hi = n if c["right"] < 0 else min(n, pos + c["right"] + 1)
    hi = max(0, hi)
    lo = 0 if c["left"] < 0 else min(hi, max(0, pos - c["left"]))
    return lo, hi, min(c["sinks"], lo, hi)


def work(c):
    e = 2
    if c["kind"].startswith("norm"):
        n = c["rows"] * c["C"]
        if c["kind"] == "norm_fwd":
            return {"bytes": e * 2 * n + 8 * c["rows"] + 8 * c["C"] * c["affine"], "flops": 8 * n}
        return {"bytes": e * 3 * n + 8 * c["rows"] + 12 * c["C"] * c["affine"], "flops": 14 * n}
    pairs, rows = 0, 0
    for n, start in zip(*lengths(c)):
        least, last, first = n, 0, 0
        for i in range(c["Nq"]):
            lo, hi, s = _span(c, n, start + i)
            pairs += hi - lo + s
            if hi > lo or s:
                least, last, first = min(least, lo), max(last, hi), max(first, s)
        rows += max(0, last - least) + min(first, least)     # keys that some query of the sequence sees
    q, kv = c["B"] * c["Nq"] * c["H"] * D * e, rows * c["KH"] * D * e
    table = 4 * c["buckets"] * c["H"]
    if c["kind"] == "attn_fwd":
        return {"bytes": 2 * q + 2 * kv + table + 4 * c["B"] * c["Nq"] * c["H"] * c["lse"], "flops": 4 * D * pairs * c["H"]}
    stats = 4 * c["B"] * c["Nq"] * c["H"]
    whole = c["B"] * c["Nk"] * c["KH"] * D * e
    return {"bytes": 3 * q + 2 * kv + 2 * whole + 2 * table + stats, "flops": 10 * D * pairs * c["H"]}


# --------------------------------------------------------------------------------------------------------------- inputs
def bucket_of(rel, buckets, distance, both):
    """the bucket of a key `rel` positions behind (or before) its query: exact for near ones, by equal ratios up to `distance`, then the last.
    A ratio's border lies at near * (distance / near) ** (k / steps): compared in whole numbers, since 64 bits are off beside one"""
    n = buckets // 2 if both else buckets
    first = n if both and rel > 0 else 0
    d = abs(rel) if both else max(0, -rel)
    near = n // 2
    if d < near:
        return first + d
    steps, k = n - near, 0
    while k + 1 < steps and d ** steps * near ** (k + 1) >= near ** steps * distance ** (k + 1):
        k += 1
    return first + near + k


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = TYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    if c["kind"].startswith("norm"):
        rows, C = c["rows"], c["C"]
        # rows of a residual stream: each with its own size and offset, a few channels that stick out
        x = torch.empty(rows, C, device="cuda", dtype=T)
        size = 1 + 3 * torch.rand(C, generator=g, device="cuda") ** 8
        for r in range(0, rows, 1 << 17):
            n = min(rows - r, 1 << 17)
            x[r:r + n] = (randn(n, C) * size * torch.exp2(2 * randn(n, 1).clamp(-3, 3)) + randn(n, 1)).to(T)
        s = {"x": x, "eps": 1e-5}
        if c["affine"]:
            s["gamma"], s["beta"] = 1 + 0.2 * randn(C), 0.1 * randn(C)
        else:
            s["gamma"] = s["beta"] = None
        if c["kind"] == "norm_bwd":
            s["dy"] = torch.empty(rows, C, device="cuda", dtype=T)
            for r in range(0, rows, 1 << 17):
                s["dy"][r:r + (1 << 17)] = (0.05 * randn(min(rows - r, 1 << 17), C)).to(T)
        return s
    B, Nq, Nk, H, KH = (c[k] for k in ("B", "Nq", "Nk", "H", "KH"))
    s = {}
    peaked = 1.7 if c["scale"] == 0.125 else 0.6       # logits of a trained layer reach some tens of either sign
    if c["cache"]:
        s["q"] = (peaked * randn(B, Nq, H * D)).to(T)
        s["k"] = torch.empty(B, Nk, KH * D, device="cuda", dtype=T)
        s["v"] = torch.empty(B, Nk, KH * D, device="cuda", dtype=T)
        for b in range(B):
            s["k"][b] = randn(Nk, KH * D).to(T)
            s["v"][b] = randn(Nk, KH * D).to(T)
    else:       # slices of the fused projection's output
        qkv = randn(B, Nq, (H + 2 * KH) * D)
        qkv[:, :, :H * D] *= peaked
        qkv = qkv.to(T)
        s["q"], s["k"], s["v"] = qkv[:, :, :H * D], qkv[:, :, H * D:(H + KH) * D], qkv[:, :, (H + KH) * D:]
    lens, starts = lengths(c)
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if c["buckets"]:
        s["table"] = randn(c["buckets"], H)
    if c["kind"] == "attn_bwd":
        s["do"] = (0.1 * randn(B, Nq, H * D)).to(T)
    return s


def _buckets(c):
    R = c["distance"]
    return torch.tensor([bucket_of(r, c["buckets"], R, c["both"]) for r in range(-R, R + 1)], dtype=torch.int64, device="cuda")


def prepare(c, seed):
    s = _inputs(c, seed)
    s["case"] = c
    if not own:
        if c["kind"] == "norm_bwd":
            x = s["x"].float()
            mean = x.mean(1, keepdim=True)
            var = (x - mean).square_().mean(1, keepdim=True)
            s["mean"], s["rstd"] = mean, 1 / torch.sqrt(var + s["eps"])
        elif c.get("buckets"):
            s["buckets"] = _buckets(c)
        return s
    from star_amd import lib
    ctx = s["ctx"] = lib.Context(0, TYPES[c["dtype"]])
    if c["kind"].startswith("norm"):
        if c["kind"] == "norm_bwd":
            s["stats"] = ctx.layer_norm_train(s["x"], s["gamma"], s["beta"], eps=s["eps"])[1]
        return s
    a = s["args"] = {"heads": c["H"], "kv_heads": c["KH"], "scale": c["scale"], "window": (c["left"], c["right"]), "sinks": c["sinks"],
                     "q_start": s["q_start"], "kv_len": s["kv_len"]}
    if c["buckets"]:
        a["bias"] = (s["table"], ctx.rel_buckets(c["buckets"], c["distance"], bidirectional=c["both"]))
    if c["kind"] == "attn_bwd":
        s["lse"] = ctx.pos_attention(s["q"], s["k"], s["v"], return_lse=True, **a)[1]
    return s


# ------------------------------------------------------------------------------------------------------------ plain form
def _norm_plain(s):
    c = s["case"]
    T = s["x"].dtype
    if c["kind"] == "norm_fwd":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        x = x - mean
        rstd = 1 / torch.sqrt(x.square().mean(1, keepdim=True) + s["eps"])
        y = x * rstd
        if c["affine"]:
            y = y * s["gamma"] + s["beta"]
        return y.to(T), torch.cat([mean, rstd], 1)
    x, dy = s["x"].float(), s["dy"].float()
    xh = (x - s["mean"]) * s["rstd"]
    dg = dy * s["gamma"] if c["affine"] else dy
    dx = (s["rstd"] * (dg - dg.mean(1, keepdim=True) - xh * (dg * xh).mean(1, keepdim=True))).to(T)
    if not c["affine"]:
        return dx
    return dx, (dy * xh).sum(0), dy.sum(0)


def _attn_plain(s):
    c = s["case"]
    B, Nq, Nk, H, KH = (c[k] for k in ("B", "Nq", "Nk", "H", "KH"))
    G = H // KH
    q, k, v, do = (s[n].float().reshape(B, -1, KH, s[n].shape[2] // KH // D, D).permute(0, 2, 3, 1, 4) if n in s else None for n in ("q", "k", "v", "do"))
    j = torch.arange(Nk, device="cuda")
    p = s["q_start"].long()[:, None, None] + torch.arange(Nq, device="cuda")[None, :, None]
    shown = (j < s["kv_len"][:, None, None]).expand(B, Nq, Nk)
    if c["right"] >= 0:
        shown = shown & (j <= p + c["right"])
    if c["left"] >= 0:
        shown = shown & ((j >= p - c["left"]) | (j < c["sinks"]))
    T = s["q"].dtype
    outs = [torch.empty(B, KH, G, Nq, D, device="cuda"), torch.empty(B, KH, G, Nq, device="cuda")]
    grads = [torch.empty(B, KH, G if n == "q" else 1, Nq if n == "q" else Nk, D, device="cuda") for n in "qkv"] if do is not None else None
    dt = torch.zeros(max(1, c["buckets"]), KH, G, device="cuda", dtype=torch.float64)
    # sequences and kv heads at a time, so that the scores of a step fit beside the rest
    nb = max(1, min(B, (1 << 29) // (H * Nq * Nk)))
    nh = max(1, min(KH, (1 << 29) // (G * Nq * Nk)))
    for b, h in ((slice(b, b + nb), slice(h, h + nh)) for b in range(0, B, nb) for h in range(0, KH, nh)):
        see = shown[b, None, None]
        qs, ks, vs = q[b, h].contiguous(), k[b, h].contiguous(), v[b, h].contiguous()
        n, m = qs.shape[:2]
        w = torch.matmul(qs.reshape(n, m, G * Nq, D), ks[:, :, 0].transpose(2, 3)).reshape(n, m, G, Nq, Nk).mul_(c["scale"])
        if c["buckets"]:
            bucket = s["buckets"][(j - p[b]).clamp(-c["distance"], c["distance"]) + c["distance"]]
            w += s["table"].reshape(-1, KH, G)[:, h][bucket].permute(0, 3, 4, 1, 2)
        w.masked_fill_(~see, -math.inf)
        dead = ~see.any(4, keepdim=True)
        most = w.amax(4, keepdim=True).masked_fill(dead, 0)
        w -= most
        w.exp_()
        total = w.sum(4, keepdim=True)
        w /= total.masked_fill(dead, 1)
        w = w.reshape(n, m, G * Nq, Nk)
        if do is None:
            outs[0][b, h] = torch.matmul(w, vs[:, :, 0]).reshape(n, m, G, Nq, D)
            outs[1][b, h] = (most + total.log())[..., 0]
            continue
        dos = do[b, h].reshape(n, m, G * Nq, D)
        grads[2][b, h, 0] = torch.matmul(w.transpose(2, 3), dos)
        dw = torch.matmul(dos, vs[:, :, 0].transpose(2, 3))
        dw -= (w * dw).sum(3, keepdim=True)
        dw *= w
        if c["buckets"]:
            # one sum for each relative position: rows turned over and padded by their count slide by one against each other, and the
            # diagonals become columns
            d = torch.nn.functional.pad(dw.reshape(n, m * G, Nq, Nk).flip(2), (0, Nq)).flatten(2)[:, :, :-Nq]
            d = d.reshape(n, m * G, Nq, Nq + Nk - 1).sum(2, dtype=torch.float64)
            gap = torch.arange(1 - Nq, Nk, device="cuda") - s["q_start"][b].long()[:, None]
            which = s["buckets"][gap.clamp(-c["distance"], c["distance"]) + c["distance"]]
            part = torch.zeros(c["buckets"], m * G, device="cuda", dtype=torch.float64)
            dt[:, h] += part.index_add_(0, which.flatten(), d.transpose(1, 2).flatten(0, 1)).reshape(-1, m, G)
        grads[0][b, h] = torch.matmul(dw, ks[:, :, 0]).mul_(c["scale"]).reshape(n, m, G, Nq, D)
        grads[1][b, h, 0] = torch.matmul(dw.transpose(2, 3), qs.reshape(n, m, G * Nq, D)).mul_(c["scale"])
    flat = lambda t: t.permute(0, 3, 1, 2, 4).reshape(B, t.shape[3], -1).to(T)  # noqa: E731
    if do is None:
        return (flat(outs[0]), outs[1].reshape(B, H, Nq)) if c["lse"] else flat(outs[0])
    grads = [flat(t) for t in grads]
    return grads + [dt.reshape(-1, H).float()] if c["buckets"] else grads


def run(s):
    c = s["case"]
    if not own:
        return _norm_plain(s) if c["kind"].startswith("norm") else _attn_plain(s)
    ctx = s["ctx"]
    if c["kind"] == "norm_fwd":
        return ctx.layer_norm_train(s["x"], s["gamma"], s["beta"], eps=s["eps"])
    if c["kind"] == "norm_bwd":
        dx, dgamma, dbeta = ctx.layer_norm_backward(s["dy"], s["x"], s["stats"], s["gamma"])
        return (dx, dgamma, dbeta) if c["affine"] else dx
    if c["kind"] == "attn_fwd":
        return ctx.pos_attention(s["q"], s["k"], s["v"], return_lse=c["lse"], **s["args"])
    dq, dk, dv, dtable = ctx.pos_attention_backward(s["do"], s["q"], s["k"], s["v"], s["lse"], **s["args"])
    return [dq, dk, dv, dtable] if c["buckets"] else [dq, dk, dv]


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def exact(c, seed):
    s = _inputs(c, seed)
    f = torch.float64
    if c["kind"].startswith("norm"):
        rows, C = s["x"].shape
        ys, stats, sums = [], [], torch.zeros(2, C, dtype=f, device="cuda")
        gamma = s["gamma"].to(f) if c["affine"] else torch.ones(C, dtype=f, device="cuda")
        for r in range(0, rows, 1 << 16):
            x = s["x"][r:r + (1 << 16)].to(f)
            var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            xh = (x - mean) / torch.sqrt(var + s["eps"])
            if c["kind"] == "norm_fwd":
                ys.append(xh * gamma + s["beta"].to(f) if c["affine"] else xh)
                stats.append(torch.cat([mean, 1 / torch.sqrt(var + s["eps"])], 1))
                continue
            dy = s["dy"][r:r + (1 << 16)].to(f)
            a = gamma * dy
            # d/dx of (x - mean) / sigma: the part along ones and the part along xh leave the row
            ys.append((a - a.sum(1, keepdim=True) / C - xh * ((a * xh).sum(1, keepdim=True) / C)) / torch.sqrt(var + s["eps"]))
            sums[0] += (dy * xh).sum(0)
            sums[1] += dy.sum(0)
        y = torch.cat(ys)
        if c["kind"] == "norm_fwd":
            return y, torch.cat(stats)
        return (y, sums[0], sums[1]) if c["affine"] else y
    if c["B"] * c["H"] > 2000:
        return None
    B, Nq, Nk, H, KH = (c[k] for k in ("B", "Nq", "Nk", "H", "KH"))
    lens, starts = lengths(c)
    out = torch.zeros(B, Nq, H, D, dtype=f, device="cuda")
    norm = torch.full((B, H, Nq), -math.inf, dtype=f, device="cuda")
    gq = torch.zeros(B, Nq, H, D, dtype=f, device="cuda") if c["kind"] == "attn_bwd" else None
    gk, gv = (torch.zeros(B, Nk, KH, D, dtype=f, device="cuda") if gq is not None else None for _ in range(2))
    gt = torch.zeros(max(1, c["buckets"]), H, dtype=f, device="cuda")
    if c["buckets"]:
        # the bucket by relative position, over every position that occurs
        far = max(max(abs(st), abs(st + Nq - 1)) for st in starts) + Nk
        cap = min(far, c["distance"])
        by_rel = torch.tensor([bucket_of(r, c["buckets"], c["distance"], c["both"]) for r in range(-cap, cap + 1)], device="cuda")
    for b in range(B):
        n = lens[b]
        for r in range(0, Nq, 2048):
            pos = torch.arange(r, min(Nq, r + 2048), device="cuda") + starts[b]
            first, last = int(pos[0]), int(pos[-1])
            lo, hi, _ = _span(c, n, first)
            hi = max(hi, _span(c, n, last)[1])
            keys = torch.arange(n, device="cuda")
            keys = keys[((keys >= lo) | (keys < c["sinks"])) & (keys < hi)]
            if not keys.numel():
                continue
            gap = keys[None, :] - pos[:, None]
            see = torch.ones_like(gap, dtype=torch.bool)
            if c["left"] >= 0:
                see &= (gap >= -c["left"]) | (keys < c["sinks"])[None, :]
            if c["right"] >= 0:
                see &= gap <= c["right"]
            some = see.any(1, keepdim=True)
            if c["buckets"]:
                which = by_rel[gap.clamp(-cap, cap) + cap]
            for h in range(H):
                kv = h * KH // H
                qh = s["q"][b, r:r + 2048, h * D:(h + 1) * D].to(f)
                kh = s["k"][b, :, kv * D:(kv + 1) * D][keys].to(f)
                vh = s["v"][b, :, kv * D:(kv + 1) * D][keys].to(f)
                logit = c["scale"] * (qh @ kh.T)
                if c["buckets"]:
                    logit += s["table"].to(f)[:, h][which]
                logit = torch.where(see, logit, torch.full_like(logit, -1e300))
                peak = logit.max(1, keepdim=True).values
                z = torch.exp(logit - peak) * see
                norm[b, h, r:r + 2048] = torch.where(some, peak + torch.log(z.sum(1, keepdim=True)), torch.full_like(peak, -math.inf))[:, 0]
                prob = torch.where(some, z / z.sum(1, keepdim=True).clamp_min(1e-300), torch.zeros_like(z))
                o = prob @ vh
                out[b, r:r + 2048, h] = o
                if gq is None:
                    continue
                g = s["do"][b, r:r + 2048, h * D:(h + 1) * D].to(f)
                gl = prob * (g @ vh.T - (g * o).sum(1, keepdim=True))
                gq[b, r:r + 2048, h] = c["scale"] * (gl @ kh)
                gk[b, :, kv].index_add_(0, keys, c["scale"] * (gl.T @ qh))
                gv[b, :, kv].index_add_(0, keys, prob.T @ g)
                if c["buckets"]:
                    for e in range(c["buckets"]):
                        gt[e, h] += gl[which == e].sum()
    if gq is None:
        return (out.reshape(B, Nq, H * D), norm) if c["lse"] else out.reshape(B, Nq, H * D)
    grads = [gq.reshape(B, Nq, H * D), gk.reshape(B, Nk, KH * D), gv.reshape(B, Nk, KH * D)]
    return grads + [gt] if c["buckets"] else grads
