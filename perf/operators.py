"""The sequence-layer and scoring operators of deepchopper_amd.ops as measurable cases.

Three operators of a recurrent genomic-language-model layer and of its answers:

  logprobs  log probabilities of given tokens (labels, bases, k-mers), entropy, top alternatives; gradient of the logits
  scan      h_t = sigmoid(f_t) h_{t-1} + (1 - sigmoid(f_t)) x_t over ragged or dense batches of reads, either direction; gradients
  norm      r' = r + scale * act(gate) * norm(y), n = norm(r'): what stands between two blocks; gradients

With `own` false, `run` is the plain form of each in elementary 32-bit torch operations; with `own` true, the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOKENS = {"i8": torch.int8, "u8": torch.uint8, "i32": torch.int32, "i64": torch.int64}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "u8": 1, "i32": 4, "i64": 8}
IGNORE = -100
EPS = 1e-5


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # a predict batch, 2 048 reads of 1 kb with [SEP]: how sure the two-class head is of every base; a quarter left padding
        {"name": "labels_of_a_batch", "op": "logprobs", "rows": 2048 * 1001, "classes": 2, "dtype": "f32", "tokens": "i8", "top": 1,
         "ignored": 0.25, "masked": False, "grad": False},
        # next-base training over the 16-row vocabulary, 64 reads of 8 k tokens
        {"name": "bases_train", "op": "logprobs", "rows": 64 * 8193, "classes": 16, "dtype": "f32", "tokens": "i8", "top": 0, "ignored": 0.1,
         "masked": False, "grad": True},
        # hexamer vocabulary (4^6), training with the entropy and a few alternatives reported
        {"name": "hexamers_train", "op": "logprobs", "rows": 16384, "classes": 4096, "dtype": "bf16", "tokens": "i32", "top": 4, "ignored": 0.02,
         "masked": False, "grad": True},
        # one serving step of a few streams over a wide, odd vocabulary, some tokens forbidden, 20 alternatives
        {"name": "wide_step", "op": "logprobs", "rows": 5, "classes": 50257, "dtype": "f16", "tokens": "i64", "top": 20, "ignored": 0.0,
         "masked": True, "grad": False},
        # training over a wide, odd vocabulary
        {"name": "wide_train", "op": "logprobs", "rows": 4096, "classes": 100003, "dtype": "bf16", "tokens": "i64", "top": 0, "ignored": 0.02,
         "masked": False, "grad": True},
        # 64 reads streamed base by base: one token of each, with the carried state
        {"name": "scan_step", "op": "scan", "seqs": 64, "short": 1, "long": 1, "channels": 256, "dtype": "bf16", "strided": False, "reverse": False,
         "grad": False},
        # the 500 - 1 500 base reads of a predict launch, packed, through one layer of the model's width
        {"name": "scan_reads", "op": "scan", "seqs": 1024, "short": 500, "long": 1500, "channels": 256, "dtype": "bf16", "strided": True,
         "reverse": False, "grad": False},
        # one read three times as long as the long convolution's positions, trained
        {"name": "scan_long_train", "op": "scan", "seqs": 1, "short": 100001, "long": 100001, "channels": 256, "dtype": "f32", "strided": False,
         "reverse": False, "grad": True},
        # a ragged nanopore-like batch trained from the 3' end, the two inputs halves of one projection
        {"name": "scan_ragged_train", "op": "scan", "seqs": 255, "short": 20, "long": 4001, "channels": 768, "dtype": "f16", "strided": True,
         "reverse": True, "grad": True},
        # between two blocks while streaming: 16 reads, one token each
        {"name": "norm_step", "op": "norm", "rows": 16, "width": 256, "dtype": "f32", "residual": "f32", "kind": "layer", "act": "sigmoid",
         "strided": False, "grad": False},
        # between two blocks of a long batch at the model's width: bf16 activations on an fp32 residual stream
        {"name": "norm_batch", "op": "norm", "rows": 524288, "width": 256, "dtype": "bf16", "residual": "f32", "kind": "layer", "act": "sigmoid",
         "strided": True, "grad": False},
        # training, a wider odd layer
        {"name": "norm_train", "op": "norm", "rows": 65537, "width": 1000, "dtype": "bf16", "residual": "bf16", "kind": "rms", "act": "silu",
         "strided": False, "grad": True},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprobs", "scan", "norm"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "logprobs":
        classes = _spread(rng, 2, 100003)
        grad = rng.random() < 0.5
        rows = _spread(rng, 1, min(2048 * 1001, 200_000_000 // classes))
        return {"op": op, "rows": rows, "classes": classes, "dtype": dtype, "tokens": rng.choice(["i8", "i32", "i64"]) if classes < 128 else rng.choice(["i32", "i64"]),
                "top": 0 if rows * classes > 80_000_000 else min(classes, rng.choice([0, 1, 2, 5, 8, 20])), "ignored": rng.choice([0.0, 0.1, 0.3]),
                "masked": rng.random() < 0.3, "grad": grad}
    if op == "scan":
        channels = _spread(rng, 16, 2048)
        grad = rng.random() < 0.5
        if rng.random() < 0.2:  # streaming: a token or a few of each read
            n = rng.choice([1, 1, 2, 7])
            return {"op": op, "seqs": _spread(rng, 1, 2048), "short": n, "long": n, "channels": channels, "dtype": dtype, "strided": rng.random() < 0.5,
                    "reverse": False, "grad": False}
        long = _spread(rng, 30, 100001)
        seqs = _spread(rng, 1, max(1, 100_000_000 // (long * channels)))
        return {"op": op, "seqs": seqs, "short": long if seqs == 1 else rng.randint(1, long), "long": long, "channels": channels, "dtype": dtype,
                "strided": rng.random() < 0.5, "reverse": rng.random() < 0.4, "grad": grad}
    width = _spread(rng, 32, 4096)
    return {"op": op, "rows": _spread(rng, 1, min(524288, 60_000_000 // width)), "width": width, "dtype": dtype, "residual": rng.choice(["f32", dtype]),
            "kind": rng.choice(["layer", "rms"]), "act": rng.choice(["identity", "sigmoid", "silu"]), "strided": rng.random() < 0.5, "grad": rng.random() < 0.5}


def _lengths(case):
    """The reads' lengths: spread evenly between the shortest and the longest, so that their sum goes by the case alone."""
    n = case["seqs"]
    return [case["long"]] if n == 1 else [case["short"] + (case["long"] - case["short"]) * i // (n - 1) for i in range(n)]


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).add_(shift).to(dtype)

    state = dict(case)
    if case["op"] == "logprobs":
        n, v = case["rows"], case["classes"]
        z = normal(n, v, scale=3.0, dtype=dt)  # a trained model's logits: a few classes far above the others
        if case["masked"]:
            z[torch.rand((n, v), generator=gen, device="cuda") < 0.2] = -math.inf  # forbidden classes
            z[n // 2:n // 2 + n // 64] = -math.inf  # rows where nothing is allowed
        t = torch.randint(0, v, (n,), generator=gen, device="cuda")
        t[torch.rand(n, generator=gen, device="cuda") < case["ignored"]] = IGNORE
        state.update(logits=z, given=t.to(TOKENS[case["tokens"]]), g_logprob=normal(n), g_entropy=normal(n, scale=0.1))
    elif case["op"] == "scan":
        lens = _lengths(case)
        random.Random(seed).shuffle(lens)
        offsets = torch.tensor([0] + lens).cumsum(0).cuda()
        total, c = sum(lens), case["channels"]
        both = torch.empty(total, 2 * c, dtype=dt, device="cuda")
        both[:, :c] = normal(total, c, dtype=dt)
        both[:, c:] = normal(total, c, scale=2.0, shift=3.0, dtype=dt)  # gates that mostly keep: memories of a few to thousands of bases
        x, f = both[:, :c], both[:, c:]
        if not case["strided"]:
            x, f = x.contiguous(), f.contiguous()
        state.update(x=x, f=f, offsets=offsets, total=total, h0=normal(case["seqs"], c))
        if case["grad"]:
            state.update(g_y=normal(total, c, dtype=dt), g_last=normal(case["seqs"], c))
    else:
        n, d = case["rows"], case["width"]
        rt = DTYPES[case["residual"]]
        both = torch.empty(n, 2 * d, dtype=dt, device="cuda")
        both[:, :d] = normal(n, d, shift=0.3, dtype=dt)
        both[:, d:] = normal(n, d, dtype=dt)
        y, gate = both[:, :d], both[:, d:]
        if not case["strided"]:
            y, gate = y.contiguous(), gate.contiguous()
        layer = case["kind"] == "layer"
        state.update(y=y, gate=gate, residual=normal(n, d, scale=2.0, dtype=rt), scale=normal(d, scale=0.1, shift=0.5),
                     post_weight=normal(d, scale=0.1, shift=1.0), post_bias=normal(d, scale=0.1) if layer else None,
                     pre_weight=normal(d, scale=0.1, shift=1.0), pre_bias=normal(d, scale=0.1) if layer else None)
        if case["grad"]:
            state.update(g_residual=normal(n, d, dtype=rt), g_normed=normal(n, d, dtype=dt))
    return state


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def _own_logprobs(s):
    from deepchopper_amd import ops

    r = ops.token_logprobs(s["logits"], s["given"], n_top=s["top"], ignore_index=IGNORE, save=s["grad"])
    out = {"logprob": r["logprob"], "entropy": r["entropy"]}
    if s["top"]:
        out.update(top_ids=r["top_ids"], top_logprob=r["top_logprob"])
    if s["grad"]:
        out["g_logits"] = ops.token_logprobs_backward(s["logits"], s["given"], r["stats"], s["g_logprob"], s["g_entropy"], ignore_index=IGNORE)
    return out


def _own_scan(s):
    from deepchopper_amd import ops

    if s["long"] == 1:  # a step: dense [reads, 1, channels]
        r = ops.gated_scan(s["x"][:, None], s["f"][:, None], h0=s["h0"])
        return {"y": r["y"][:, 0], "h_last": r["h_last"]}
    r = ops.gated_scan(s["x"], s["f"], offsets=s["offsets"], max_len=s["long"], h0=s["h0"], reverse=s["reverse"], save=s["grad"])
    out = {"y": r["y"], "h_last": r["h_last"]}
    if s["grad"]:
        g = ops.gated_scan_backward(s["x"], s["f"], r["saved"], s["g_y"], grad_h_last=s["g_last"], h0=s["h0"], offsets=s["offsets"], max_len=s["long"],
                                    reverse=s["reverse"])
        out.update(g_x=g["grad_x"], g_f=g["grad_f"], g_h0=g["grad_h0"])
    return out


def _own_norm(s):
    from deepchopper_amd import ops

    kw = dict(kind=s["kind"], gate_act=s["act"], scale=s["scale"], post_weight=s["post_weight"], post_bias=s["post_bias"],
              pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], eps=EPS)
    r = ops.block_norm(s["y"], s["residual"], s["gate"], **kw)
    out = {"residual": r["residual"], "normed": r["normed"]}
    if s["grad"]:
        g = ops.block_norm_backward(s["y"], s["residual"], s["gate"], grad_residual=s["g_residual"], grad_normed=s["g_normed"], **kw)
        names = ("y", "gate", "residual", "scale", "post_weight", "pre_weight") + (("post_bias", "pre_bias") if s["kind"] == "layer" else ())
        out.update({"g_" + k: g["grad_" + k] for k in names})
    return out


def _plain_logprobs(s):
    z, t = s["logits"].float(), s["given"].long()
    live = t != IGNORE
    at = t.clamp_min(0)[:, None]
    top = z.amax(-1, keepdim=True)
    some = top > -math.inf
    d = z - torch.where(some, top, 0.0)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    logp = torch.where(some, d - total.log(), -math.inf)
    p = e / torch.where(some, total, 1.0)
    entropy = -(p * torch.where(p > 0, logp, 0.0)).sum(-1)
    out = {"logprob": torch.where(live, logp.gather(1, at)[:, 0], 0.0), "entropy": torch.where(live, entropy, 0.0)}
    if s["top"]:
        ids = z.sort(dim=-1, descending=True, stable=True).indices[:, :s["top"]]
        out["top_ids"] = torch.where(live[:, None], ids, -1).int()
        out["top_logprob"] = torch.where(live[:, None], logp.gather(1, ids), 0.0)
    if s["grad"]:
        gl, gh = (torch.where(live, s[k], 0.0)[:, None] for k in ("g_logprob", "g_entropy"))
        g = -p * (gl + gh * (torch.where(p > 0, logp, 0.0) + entropy[:, None]))
        g.scatter_add_(1, at, torch.where(some, gl, 0.0))
        out["g_logits"] = g.to(s["logits"].dtype)
    return out


def _doubling(a, b, longest):
    """h_t = a_t h_{t-1} + b_t along the first axis, by doubling; a is 0 where a read begins, so nothing passes from read to read."""
    step = 1
    while step < longest:
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_scan(s):
    x, f, offsets, h0 = s["x"].float(), s["f"].float(), s["offsets"], s["h0"]
    first, last = offsets[:-1], offsets[1:] - 1
    if s["reverse"]:
        x, f = x.flip(0), f.flip(0)
        first, last = s["total"] - 1 - last, s["total"] - 1 - first
    a, w = f.sigmoid(), (-f).sigmoid()
    kept = a.index_fill(0, first, 0.0)
    b = w * x
    b[first] += a[first] * h0
    h = _doubling(kept, b, s["long"])
    y = h.flip(0) if s["reverse"] else h
    out = {"y": y.to(s["x"].dtype), "h_last": h[last]}
    if s["grad"]:
        g = s["g_y"].float()
        g = g.flip(0) if s["reverse"] else g.clone()
        g[last] += s["g_last"]
        onward = torch.cat([kept[1:], torch.zeros_like(kept[:1])])  # what passes from t + 1 back to t
        g = _doubling(onward.flip(0), g.flip(0), s["long"]).flip(0)
        before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
        before[first] = h0
        gx, gf = g * w, g * (before - x) * a * w
        if s["reverse"]:
            gx, gf = gx.flip(0), gf.flip(0)
        out.update(g_x=gx.to(s["x"].dtype), g_f=gf.to(s["f"].dtype), g_h0=a[first] * g[first])
    return out


def _normalise(x, kind):
    """(x - mean) / deviation, or x / root mean square, and the factor."""
    c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    factor = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return c * factor, factor


def _normalise_back(g, hat, factor, kind):
    g = g - hat * (g * hat).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return factor * g


def _plain_norm(s):
    kind, act = s["kind"], s["act"]
    y, gate, r = s["y"].float(), s["gate"].float(), s["residual"].float()
    hat, factor = _normalise(y, kind)
    u = hat * s["post_weight"] + (s["post_bias"] if kind == "layer" else 0.0)
    sig = gate.sigmoid()
    a = gate if act == "identity" else sig if act == "sigmoid" else gate * sig
    v = a * u
    r2 = r + s["scale"] * v
    hat2, factor2 = _normalise(r2, kind)
    n = hat2 * s["pre_weight"] + (s["pre_bias"] if kind == "layer" else 0.0)
    out = {"residual": r2.to(s["residual"].dtype), "normed": n.to(s["y"].dtype)}
    if s["grad"]:
        gn = s["g_normed"].float()
        t = s["g_residual"].float() + _normalise_back(gn * s["pre_weight"], hat2, factor2, kind)
        gv = t * s["scale"]
        slope = torch.ones_like(sig) if act == "identity" else sig * (1 - sig) if act == "sigmoid" else sig * (1 + gate * (1 - sig))
        gu = gv * a
        out.update(g_y=_normalise_back(gu * s["post_weight"], hat, factor, kind).to(s["y"].dtype), g_gate=(gv * u * slope).to(s["gate"].dtype),
                   g_residual=t.to(s["residual"].dtype), g_scale=(t * v).sum(0), g_post_weight=(gu * hat).sum(0), g_pre_weight=(gn * hat2).sum(0))
        if kind == "layer":
            out.update(g_post_bias=gu.sum(0), g_pre_bias=gn.sum(0))
    return out


_OWN = {"logprobs": _own_logprobs, "scan": _own_scan, "norm": _own_norm}
_PLAIN = {"logprobs": _plain_logprobs, "scan": _plain_scan, "norm": _plain_norm}


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    es = SIZE[case["dtype"]]
    if case["op"] == "logprobs":
        n, v = case["rows"], case["classes"]
        live = n * (1.0 - case["ignored"])  # a row without a token is not read
        b = live * v * es + n * (SIZE[case["tokens"]] + 8 + 8 * case["top"])
        fl = live * v * 6.0
        if case["grad"]:
            b += n * v * es + n * 8
            fl += live * v * 8.0
        return {"bytes": b, "flops": fl}
    if case["op"] == "scan":
        n, c, k = sum(_lengths(case)), case["channels"], case["seqs"]
        b = 3 * n * c * es + 2 * k * c * 4 + 8 * (k + 1)
        fl = 10.0 * n * c
        if case["grad"]:
            b += 3 * n * c * es + 2 * k * c * 4
            fl += 16.0 * n * c
        return {"bytes": b, "flops": fl}
    n, d, rs = case["rows"], case["width"], SIZE[case["residual"]]
    vectors = 5 if case["kind"] == "layer" else 3
    b = n * d * (3 * es + 2 * rs) + vectors * d * 4
    fl = 20.0 * n * d
    if case["grad"]:
        b += n * d * (3 * es + 2 * rs) + vectors * d * 4
        fl += 40.0 * n * d
    return {"bytes": b, "flops": fl}


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](s)


def _exact_logprobs(s):
    n, v, parts = s["rows"], s["classes"], []
    block = max(1, 200_000_000 // v)
    for r0 in range(0, n, block):  # rows in blocks: 64-bit copies of the whole would not always fit
        z = s["logits"][r0:r0 + block].double()
        t = s["given"][r0:r0 + block].long()
        live, idx = t != IGNORE, torch.arange(z.shape[0], device=z.device)
        lse = torch.logsumexp(z, -1, keepdim=True)
        empty = lse == -math.inf
        logp = torch.where(empty, -math.inf, z - lse.masked_fill(empty, 0.0))
        p = logp.exp()
        h = -torch.special.xlogy(p, p).sum(-1)
        at = t.masked_fill(~live, 0)
        part = {"logprob": logp[idx, at].masked_fill(~live, 0.0), "entropy": h.masked_fill(~live, 0.0)}
        if s["top"]:
            ids, taken = [], torch.zeros_like(z, dtype=torch.bool)
            for _ in range(s["top"]):
                best = z.masked_fill(taken, -math.inf).amax(-1, keepdim=True)
                pick = torch.where(~taken & (z == best), torch.arange(v, device=z.device), v).amin(-1)
                taken[idx, pick] = True
                ids.append(pick)
            ids = torch.stack(ids, -1)
            part["top_ids"] = ids.masked_fill(~live[:, None], -1).int()
            part["top_logprob"] = logp.gather(1, ids).masked_fill(~live[:, None], 0.0)
        if s["grad"]:
            gl, gh = s["g_logprob"][r0:r0 + block].double(), s["g_entropy"][r0:r0 + block].double()
            g = p * -gl[:, None] - gh[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
            g[idx, at] += gl
            part["g_logits"] = g.masked_fill((~live | empty[:, 0])[:, None], 0.0)
        parts.append(part)
    return {k: torch.cat([q[k] for q in parts]) for k in parts[0]}


def _exact_scan(s):
    """One token of every read after the other."""
    lens = s["offsets"].diff().tolist()
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    starts = s["offsets"][:-1][torch.tensor(order, device="cuda")]
    ends = s["offsets"][1:][torch.tensor(order, device="cuda")]
    lens = [lens[i] for i in order]
    longest, back = lens[0], s["reverse"]
    if longest > 150000:
        return None
    alive, k = [], len(lens)
    for t in range(longest):
        while lens[k - 1] <= t:
            k -= 1
        alive.append(k)
    x, f = s["x"].double(), s["f"].double()
    y, before = torch.empty_like(x), torch.empty_like(x) if s["grad"] else None
    h = s["h0"].double()[torch.tensor(order, device="cuda")]
    for t in range(longest):
        k = alive[t]
        at = ends[:k] - 1 - t if back else starts[:k] + t
        a = 1.0 / (1.0 + torch.exp(-f[at]))
        if before is not None:
            before[at] = h[:k]
        h[:k] = x[at] + a * (h[:k] - x[at])
        y[at] = h[:k]
    place = torch.empty(len(order), dtype=torch.long, device="cuda")
    place[torch.tensor(order, device="cuda")] = torch.arange(len(order), device="cuda")
    out = {"y": y, "h_last": h[place]}
    if s["grad"]:
        g = s["g_last"].double()[torch.tensor(order, device="cuda")]
        gy, gx, gf = s["g_y"], torch.empty_like(x), torch.empty_like(x)
        for t in reversed(range(longest)):
            k = alive[t]
            at = ends[:k] - 1 - t if back else starts[:k] + t
            a = 1.0 / (1.0 + torch.exp(-f[at]))
            total = g[:k] + gy[at].double()
            gx[at] = total * (1 - a)
            gf[at] = total * (before[at] - x[at]) * a * (1 - a)
            g[:k] = total * a
        out.update(g_x=gx, g_f=gf, g_h0=g[place])
    return out


def _exact_norm(s):
    """The outputs from torch's own 64-bit arithmetic, the gradients by differentiating them, in blocks of rows."""
    layer, d = s["kind"] == "layer", s["width"]
    block = max(1, 30_000_000 // d)
    vectors = {k: s[k].double().requires_grad_(s["grad"]) for k in ("scale", "post_weight", "pre_weight") + (("post_bias", "pre_bias") if layer else ())}
    parts = []
    for r0 in range(0, s["rows"], block):
        ins = {k: s[k][r0:r0 + block].double().requires_grad_(s["grad"]) for k in ("y", "gate", "residual")}

        def norm(v, w, b):
            if layer:
                var, mean = torch.var_mean(v, -1, keepdim=True, unbiased=False)
                return (v - mean) / (var + EPS).sqrt() * w + b
            return v / ((v * v).sum(-1, keepdim=True) / d + EPS).sqrt() * w

        u = norm(ins["y"], vectors["post_weight"], vectors.get("post_bias"))
        gate = ins["gate"]
        if s["act"] != "identity":
            gate = (gate if s["act"] == "silu" else 1.0) / (1.0 + torch.exp(-gate))
        r = ins["residual"] + vectors["scale"] * (gate * u)
        n = norm(r, vectors["pre_weight"], vectors.get("pre_bias"))
        part = {"residual": r.detach(), "normed": n.detach()}
        if s["grad"]:
            torch.autograd.backward([r, n], [s["g_residual"][r0:r0 + block].double(), s["g_normed"][r0:r0 + block].double()])
            part.update({"g_" + k: v.grad for k, v in ins.items()})
        parts.append(part)
    out = {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
    if s["grad"]:
        out.update({"g_" + k: v.grad for k, v in vectors.items()})
    return out
