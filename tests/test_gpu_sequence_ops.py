"""GPU tests of the sequence-layer and scoring operators (gated_scan, block_norm, token_logprobs) against their definitions in 64 bits.

A floating output may be off by the oracle's bound for 32-bit arithmetic plus half a step of its own type."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}  # half the smallest step (fp32 results below 2^-126 may be flushed)


@pytest.fixture(scope="module")
def env(hip_lib):
    import torch

    from deepchopper_amd import _lib, ops

    assert _lib.device_count() >= 1, "GPU tests need a HIP device; there is no CPU fallback"
    return torch, ops


def check(name, got, want, bound):
    """got: tensor; want / bound float64 arrays of its shape."""
    dt = str(got.dtype).replace("torch.", "")
    g = got.detach().double().cpu().numpy().reshape(want.shape)
    if dt == "float16":  # beyond the type's range
        want = np.where(np.abs(want) > 65519, np.inf * np.sign(want), want)
    with np.errstate(invalid="ignore"):
        same = (g == want) | (np.isnan(g) & np.isnan(want))
        off = np.abs(g - want) - (bound + HALF_STEP[dt] * (np.abs(want) + bound) + TINY[dt])
    wrong = ~same & ~(off <= 0)
    assert not wrong.any(), f"{name}: {wrong.sum()} of {wrong.size} values off, first at {tuple(np.argwhere(wrong)[0])}: {g[wrong][:4]} for {want[wrong][:4]}"


def host(t):
    return t.detach().double().cpu().numpy()


def make(torch, gen, *shape, dtype="float32", scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen) * scale + shift).to(getattr(torch, dtype)).cuda()


# ------------------------------------------------------------------------------------------
# gated_scan
# ------------------------------------------------------------------------------------------
def scan_all(torch, ops, x, f, ranges, *, how, reverse=False, h0=None, gy=None, gl=None, max_len=None):
    """Forward and backward through the wrappers; `how`: dense, offsets or ends (begin / end)."""
    if how == "dense":
        kw = {}
        shape = (len(ranges), ranges[0][1] - ranges[0][0], x.shape[1])
        x, f, gy = x.view(shape), f.view(shape), gy.view(shape)
    elif how == "offsets":
        kw = {"offsets": torch.tensor([r[0] for r in ranges] + [ranges[-1][1]], dtype=torch.int64).cuda()}
    else:
        kw = {"begin": torch.tensor([r[0] for r in ranges], dtype=torch.int64).cuda(), "end": torch.tensor([r[1] for r in ranges], dtype=torch.int64).cuda()}
    if how != "dense" and max_len is not None:
        kw["max_len"] = max_len
    r = ops.gated_scan(x, f, h0=h0, reverse=reverse, save=True, **kw)
    g = ops.gated_scan_backward(x, f, r["saved"], gy, grad_h_last=gl, h0=h0, reverse=reverse, **kw)
    return {"y": r["y"], "h_last": r["h_last"], **g}


def check_scan(torch, ops, seed, lengths, channels, dtype, *, how="offsets", reverse=False, state=True, strided=False, max_len=None, f_scale=2.0, f_shift=1.0):
    from oracle import sequence_ref as ref

    gen = torch.Generator().manual_seed(seed)
    total, k = sum(lengths), len(lengths)
    both = make(torch, gen, total, 2 * channels + 1, dtype=dtype)
    x, f = both[:, :channels], both[:, channels + 1:]
    f.mul_(f_scale).add_(f_shift)
    if not strided:
        x, f = x.contiguous(), f.contiguous()
    ends = np.cumsum(lengths)
    ranges = [(int(e - n), int(e)) for e, n in zip(ends, lengths)]
    gy = make(torch, gen, total, channels, dtype=dtype)
    h0 = make(torch, gen, k, channels) if state else None
    gl = make(torch, gen, k, channels) if state else None
    got = scan_all(torch, ops, x, f, ranges, how=how, reverse=reverse, h0=h0, gy=gy, gl=gl, max_len=max_len)
    want, bound = ref.gated_scan(host(x), host(f), ranges, None if h0 is None else host(h0), reverse, host(gy), None if gl is None else host(gl))
    for name in want:
        check(name, got[name], want[name], bound[name])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("lengths,channels", [
    ([1], 1), ([1, 1, 1], 256), ([0, 1, 0], 3), ([7, 7], 64), ([16, 16, 16], 130), ([17, 17], 66), ([127, 128, 129], 64), ([5, 0, 300, 1, 257], 65),
    ([1000], 17), ([640, 64], 34), ([33] * 9, 16), ([2, 513, 1], 15), ([256, 255], 258)])
def test_gated_scan_matches_the_definition(env, dtype, lengths, channels):
    check_scan(*env, 1, lengths, channels, dtype)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("strided", [False, True])
def test_gated_scan_directions_states_and_strides(env, reverse, state, strided):
    check_scan(*env, 2, [130, 1, 77, 400], 48, "bfloat16", reverse=reverse, state=state, strided=strided)
    check_scan(*env, 3, [130, 1, 77, 400], 47, "float32", reverse=reverse, state=state, strided=strided)


@pytest.mark.parametrize("lengths", [[1] * 5, [4] * 3, [16] * 4, [130] * 3, [1], [700]])
@pytest.mark.parametrize("reverse", [False, True])
def test_gated_scan_dense(env, lengths, reverse):
    check_scan(*env, 4, lengths, 40, "float16", how="dense", reverse=reverse)


@pytest.mark.parametrize("reverse", [False, True])
def test_gated_scan_one_long_sequence(env, reverse):
    """Long enough to be divided over many workgroups, with gates that keep for thousands of tokens."""
    check_scan(*env, 5, [30011], 5, "float32", reverse=reverse, f_scale=2.0, f_shift=6.0)
    check_scan(*env, 6, [9001, 3, 20000], 66, "bfloat16", reverse=reverse, f_shift=4.0)


def test_gated_scan_max_len_is_only_a_bound(env):
    check_scan(*env, 7, [50, 3, 20], 33, "float32", max_len=5000)
    check_scan(*env, 7, [5, 3, 2], 33, "float32", max_len=16)


@pytest.mark.parametrize("gate", [-90.0, -30.0, 0.0, 12.0, 30.0, 90.0])
def test_gated_scan_extreme_constant_gates(env, gate):
    check_scan(*env, 8, [900, 1], 8, "float32", f_scale=0.0, f_shift=gate)


def test_gated_scan_infinite_gates_keep_and_take(env):
    """+inf keeps the state whatever stands in x (padding inside a row); -inf takes x."""
    torch, ops = env
    from oracle import sequence_ref as ref

    gen = torch.Generator().manual_seed(9)
    n, c = 300, 20
    x, f, gy = make(torch, gen, n, c), make(torch, gen, n, c), make(torch, gen, n, c)
    f[::7] = float("inf")
    f[3::11] = float("-inf")
    x[::14] = float("nan")
    x[7::14] = float("inf")
    f[::7] = float("inf")
    h0 = make(torch, gen, 1, c)
    got = scan_all(torch, ops, x, f, [(0, n)], how="offsets", h0=h0, gy=gy)
    want, bound = ref.gated_scan(host(x), host(f), [(0, n)], host(h0), False, host(gy))
    for name in want:
        check(name, got[name], want[name], bound[name])


@pytest.mark.parametrize("reverse", [False, True])
def test_gated_scan_begin_and_end(env, reverse):
    """Left-padded rows: sequences in any order with gaps; what stands in the gaps stays."""
    torch, ops = env
    from oracle import sequence_ref as ref

    gen = torch.Generator().manual_seed(10)
    n, c = 900, 36
    x, f, gy = (make(torch, gen, n, c, dtype="bfloat16") for _ in range(3))
    ranges = [(500, 900), (10, 130), (130, 131), (200, 200), (255, 385)]
    got = scan_all(torch, ops, x, f, ranges, how="ends", reverse=reverse, gy=gy)
    want, bound = ref.gated_scan(host(x), host(f), ranges, None, reverse, host(gy))
    covered = ~np.isnan(want["y"][:, 0])
    for name in want:
        if want[name].shape[0] == n:
            check(name, got[name][torch.from_numpy(covered).cuda()], want[name][covered], bound[name][covered])
            assert (host(got[name])[~covered] == 0).all()
        else:
            check(name, got[name], want[name], bound[name])
    out = torch.full((n, c), 3.0, dtype=torch.bfloat16, device="cuda")
    b, e = (torch.tensor([r[i] for r in ranges]).cuda() for i in (0, 1))
    r = ops.gated_scan(x, f, begin=b, end=e, reverse=reverse, out=out)
    assert r["y"] is out and (host(out)[~covered] == 3.0).all() and torch.equal(out[torch.from_numpy(covered).cuda()], got["y"][torch.from_numpy(covered).cuda()])


def test_gated_scan_tokens_outside_the_offsets(env):
    """Rows in front of the first and behind the last sequence: zero in what the call makes, left as they were in `out`."""
    torch, ops = env
    gen = torch.Generator().manual_seed(11)
    n, c = 400, 24
    x, f, gy = (make(torch, gen, n, c) for _ in range(3))
    off = torch.tensor([30, 160, 300]).cuda()
    out = torch.full((n, c), 7.0, device="cuda")
    kept = ops.gated_scan(x, f, offsets=off, out=out, save=True)
    made = ops.gated_scan(x, f, offsets=off, save=True)
    g = ops.gated_scan_backward(x, f, made["saved"], gy, offsets=off)
    assert torch.equal(kept["y"][30:300], made["y"][30:300])
    for t, v in ((out, 7.0), (made["y"], 0.0), (g["grad_x"], 0.0), (g["grad_f"], 0.0)):
        assert (t[:30] == v).all() and (t[300:] == v).all()
    for max_len in (0, 5000):
        none = ops.gated_scan(x, f, offsets=torch.zeros(1, dtype=torch.int64, device="cuda"), max_len=max_len)
        assert (none["y"] == 0).all() and none["h_last"].shape == (0, c)
        h0 = make(torch, gen, 3, c)
        empty = ops.gated_scan(x[:0], f[:0], offsets=torch.zeros(4, dtype=torch.int64, device="cuda"), max_len=max_len, h0=h0, save=True)
        assert torch.equal(empty["h_last"], h0)
        back = ops.gated_scan_backward(x[:0], f[:0], empty["saved"], gy[:0], grad_h_last=h0, offsets=torch.zeros(4, dtype=torch.int64, device="cuda"), max_len=max_len)
        assert torch.equal(back["grad_h0"], h0)


def test_gated_scan_streams_token_by_token(env):
    """A read in one call, and token by token with the state kept in place: the same states."""
    torch, ops = env
    gen = torch.Generator().manual_seed(12)
    b, n, c = 3, 150, 70
    x, f, h0 = make(torch, gen, b, n, c), make(torch, gen, b, n, c), make(torch, gen, b, c)
    whole = ops.gated_scan(x, f, h0=h0)
    h = h0.clone()
    for t in range(n):
        r = ops.gated_scan(x[:, t:t + 1], f[:, t:t + 1], h0=h, h_last=h)
        assert r["h_last"] is h
        assert (r["y"][:, 0] - whole["y"][:, t]).abs().max() < 2e-6 and torch.equal(r["y"][:, 0], h)
    assert (h - whole["h_last"]).abs().max() < 2e-6  # 150 steps: at most 150 x 6 x 2^-24 x 1 / 50 of memory apart


@pytest.mark.parametrize("n,c,dtype", [(3000, 33, "bfloat16"), (300, 129, "float16"), (5, 7, "bfloat16"), (3000, 64, "float32")])
def test_gated_scan_state_kept_in_place(env, n, c, dtype):
    """h_last = h0, over chunks, tiles and single tokens, odd channels included: what a state of its own gives."""
    torch, ops = env
    gen = torch.Generator().manual_seed(16)
    x, f = make(torch, gen, 2, n, c, dtype=dtype), make(torch, gen, 2, n, c, dtype=dtype, shift=4.0)
    h0 = make(torch, gen, 2, c)
    want = ops.gated_scan(x, f, h0=h0)
    for _ in range(3):
        h = h0.clone()
        got = ops.gated_scan(x, f, h0=h, h_last=h)
        assert got["h_last"] is h
        # (one channel a lane or two: the same steps, so the same bits)
        assert torch.equal(h, want["h_last"]) and torch.equal(got["y"], want["y"])


def test_gated_scan_strides_beyond_a_tile_offset(env):
    """Rows more than 2^20 elements apart: whole tiles go the checked way too."""
    from oracle import sequence_ref as ref

    torch, ops = env
    gen = torch.Generator().manual_seed(17)
    n, c = 200, 64
    wide = torch.empty((n, (1 << 20) + 8), dtype=torch.bfloat16, device="cuda")
    x, f = wide[:, :c], wide[:, c:2 * c]
    x.copy_(torch.randn((n, c), generator=gen))
    f.copy_(torch.randn((n, c), generator=gen) + 1)
    for reverse in (False, True):
        r = ops.gated_scan(x, f, offsets=torch.tensor([0, n]).cuda(), max_len=n, reverse=reverse)
        want, bound = ref.gated_scan(host(x), host(f), [(0, n)], reverse=reverse)
        check("y", r["y"], want["y"], bound["y"])


def test_gated_scan_refuses_bad_sequences_on_the_device(env):
    """A sequence outside the tokens, backwards or longer than max_len: NaN state, nothing else of it written."""
    torch, ops = env
    gen = torch.Generator().manual_seed(13)
    n, c = 600, 40
    x, f, gy = (make(torch, gen, n, c) for _ in range(3))
    b = torch.tensor([0, -5, 90, 100, 590, 300]).cuda()
    e = torch.tensor([50, 20, 80, 420, 601, 360]).cuda()
    out = torch.full((n, c), 5.0, device="cuda")
    for max_len in (200, 16 * 13, 60):
        out.fill_(5.0)
        r = ops.gated_scan(x, f, begin=b, end=e, max_len=max_len, out=out, save=True)
        bad = torch.isnan(r["h_last"]).all(1).tolist()
        assert bad == [False, True, True, True, True, False] and not torch.isnan(r["h_last"][[0, 5]]).any()
        covered = torch.zeros(n, dtype=torch.bool, device="cuda")
        covered[:50] = covered[300:360] = True
        assert (out[~covered] == 5.0).all() and (out[covered] != 5.0).any(1).all()
        g = ops.gated_scan_backward(x, f, r["saved"], gy, begin=b, end=e, max_len=max_len)
        assert torch.isnan(g["grad_h0"]).all(1).tolist() == bad and (g["grad_x"][~covered] == 0).all()


def test_gated_scan_gradients_against_differences(env):
    """d loss / d input by central differences of the kernel's own forward pass, loss = sum(y gy) + sum(h_last gl)."""
    torch, ops = env
    gen = torch.Generator().manual_seed(14)
    n, c = 40, 2
    x, f, gy = (make(torch, gen, n, c) for _ in range(3))
    h0, gl = make(torch, gen, 2, c), make(torch, gen, 2, c)
    off = torch.tensor([0, 13, n]).cuda()

    def loss(x, f, h0):
        r = ops.gated_scan(x, f, offsets=off, max_len=27, h0=h0)
        return float((r["y"].double() * gy.double()).sum() + (r["h_last"].double() * gl.double()).sum())

    saved = ops.gated_scan(x, f, offsets=off, h0=h0, save=True)["saved"]
    g = ops.gated_scan_backward(x, f, saved, gy, grad_h_last=gl, h0=h0, offsets=off)
    step = 2.0 ** -6
    for i, (t, grad) in enumerate(((x, g["grad_x"]), (f, g["grad_f"]), (h0, g["grad_h0"]))):
        for flat in range(0, t.numel(), 7):
            plus, minus = t.clone(), t.clone()
            plus.view(-1)[flat] += step
            minus.view(-1)[flat] -= step
            width = float((plus - minus).view(-1)[flat])
            args = [[x, f, h0] for _ in range(2)]
            args[0][i], args[1][i] = plus, minus
            num = (loss(*args[0]) - loss(*args[1])) / width
            # fp32 noise of the 80 terms over the step, and step^2 / 6 of a third derivative below 5
            assert abs(num - float(grad.view(-1)[flat])) < 80 * 6 * 2.0 ** -24 / width + 5 * step * step / 6


def test_gated_scan_offsets_beyond_32_bits(env):
    """Rows 65 536 elements apart: the last ones start behind element 2^32."""
    torch, ops = env
    from oracle import sequence_ref as ref

    gen = torch.Generator().manual_seed(15)
    n, c = 65800, 8
    wide = torch.empty((n, 65536), dtype=torch.bfloat16, device="cuda")
    x = wide[:, :c]
    x.copy_(torch.randn((n, c), generator=gen))
    f = wide[:, 100:100 + c]
    f.copy_(torch.randn((n, c), generator=gen) + 2)
    ranges = [(0, 65500), (65500, 65800)]
    off = torch.tensor([0, 65500, 65800]).cuda()
    out = wide[:, 200:200 + c]
    r = ops.gated_scan(x, f, offsets=off, max_len=65500, out=out)
    tail = slice(65500, n)
    want, bound = ref.gated_scan(host(x[tail]), host(f[tail]), [(0, 300)])
    check("y", r["y"][tail].contiguous(), want["y"], bound["y"])
    check("h_last", r["h_last"][1:], want["h_last"], bound["h_last"])


# ------------------------------------------------------------------------------------------
# block_norm
# ------------------------------------------------------------------------------------------
def norm_inputs(torch, gen, shape, dtype, residual, *, strided=False, gate=True, biases=True):
    w = shape[-1]
    both = make(torch, gen, *shape[:-1], 2 * w + 3, dtype=dtype, shift=0.3)
    y, g = both[..., :w], both[..., w + 3:]
    if not strided:
        y, g = y.contiguous(), g.contiguous()
    kw = dict(scale=make(torch, gen, w, scale=0.2, shift=0.5), post_weight=make(torch, gen, w, scale=0.2, shift=1.0),
              pre_weight=make(torch, gen, w, scale=0.2, shift=1.0))
    if biases:
        kw.update(post_bias=make(torch, gen, w, scale=0.2), pre_bias=make(torch, gen, w, scale=0.2))
    return y, make(torch, gen, *shape, dtype=residual, scale=2.0), g if gate else None, kw


def check_norm(torch, ops, y, r, g, kw, gr, gn, *, kind, act, post=True, pre=True):
    from oracle import sequence_ref as ref

    got = ops.block_norm(y, r, g, kind=kind, gate_act=act, post=post, pre=pre, **kw)
    back = ops.block_norm_backward(y, r, g, grad_residual=gr, grad_normed=gn, kind=kind, gate_act=act, post=post, **kw)
    h = lambda t: None if t is None else host(t)  # noqa: E731
    want, bound = ref.block_norm(h(y), h(r), h(g), kind=kind, act=act, post=post, pre=pre, **{k: h(v) for k, v in kw.items()}, grad_residual=h(gr), grad_normed=h(gn))
    seen = 0
    for name, t in {**got, **back}.items():
        if t is None or name not in want or (name == "residual" and y is None):
            continue
        check(name, t, want[name], bound[name])
        seen += 1
    return seen


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype,residual", [("float32", "float32"), ("bfloat16", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("rows,width", [(1, 256), (3, 1), (130, 8), (33, 63), (65, 65), (300, 256), (17, 257), (9, 1000), (21, 1024), (5, 2049), (3, 4096), (2, 8192)])
def test_block_norm_matches_the_definition(env, kind, dtype, residual, rows, width):
    torch, ops = env
    gen = torch.Generator().manual_seed(rows * width)
    y, r, g, kw = norm_inputs(torch, gen, (rows, width), dtype, residual, biases=kind == "layer")
    gr, gn = make(torch, gen, rows, width, dtype=residual), make(torch, gen, rows, width, dtype=dtype)
    assert check_norm(torch, ops, y, r, g, kw, gr, gn, kind=kind, act="sigmoid") >= 8


@pytest.mark.parametrize("act", ["identity", "sigmoid", "silu"])
@pytest.mark.parametrize("strided", [False, True])
def test_block_norm_gates_and_strides(env, act, strided):
    torch, ops = env
    gen = torch.Generator().manual_seed(21)
    for shape in ((4, 37, 96), (150, 97)):
        y, r, g, kw = norm_inputs(torch, gen, shape, "bfloat16", "float32", strided=strided)
        gr, gn = make(torch, gen, *shape), make(torch, gen, *shape, dtype="bfloat16")
        if strided:  # gradients of broadcast outputs: one row for all
            gr = gr[..., :1, :].expand(shape) if len(shape) == 2 else gr
            gn = gn[:1].expand(shape) if len(shape) == 2 else gn
        check_norm(torch, ops, y, r, g, kw, gr, gn, kind="layer", act=act)


@pytest.mark.parametrize("width", [64, 100, 515])
def test_block_norm_parts(env, width):
    """Every part can be left out: the first norm of a model, the last block, no gate, no residual, no post norm, no vectors."""
    torch, ops = env
    gen = torch.Generator().manual_seed(22)
    y, r, g, kw = norm_inputs(torch, gen, (70, width), "float32", "float32")
    gr, gn = make(torch, gen, 70, width), make(torch, gen, 70, width)
    pre = {k: v for k, v in kw.items() if k.startswith("pre")}
    assert check_norm(torch, ops, None, r, None, pre, gr, gn, kind="layer", act="identity") == 4
    check_norm(torch, ops, y, r, None, kw, gr, gn, kind="layer", act="identity")
    check_norm(torch, ops, y, None, g, kw, gr, gn, kind="rms", act="silu")
    check_norm(torch, ops, y, r, g, {k: v for k, v in kw.items() if "post" not in k}, gr, gn, kind="layer", act="sigmoid", post=False)
    check_norm(torch, ops, y, r, g, {}, gr, gn, kind="layer", act="sigmoid")
    check_norm(torch, ops, y, r, g, kw, gr, None, kind="layer", act="sigmoid")
    check_norm(torch, ops, y, r, g, kw, None, gn, kind="layer", act="sigmoid")
    last = ops.block_norm(y, r, g, pre=False, **{k: v for k, v in kw.items() if not k.startswith("pre")})
    assert last["normed"] is None and torch.equal(last["residual"], ops.block_norm(y, r, g, **kw)["residual"])


def test_block_norm_in_place_and_repeatable(env):
    torch, ops = env
    gen = torch.Generator().manual_seed(23)
    y, r, g, kw = norm_inputs(torch, gen, (5000, 256), "bfloat16", "float32")
    gr, gn = make(torch, gen, 5000, 256), make(torch, gen, 5000, 256, dtype="bfloat16")
    a = ops.block_norm(y, r, g, **kw)
    b = [ops.block_norm_backward(y, r, g, grad_residual=gr, grad_normed=gn, **kw) for _ in range(3)]
    for k in b[0]:
        assert torch.equal(b[0][k], b[1][k]) and torch.equal(b[0][k], b[2][k]), k
    inside = r.clone()
    c = ops.block_norm(y, inside, g, out=inside, **kw)
    assert c["residual"] is inside and torch.equal(inside, a["residual"]) and torch.equal(c["normed"], a["normed"])


def test_block_norm_far_mean_and_constant_rows(env):
    """A mean thousands of deviations away, rows of one value, rows of zeros."""
    torch, ops = env
    gen = torch.Generator().manual_seed(24)
    y, r, g, kw = norm_inputs(torch, gen, (40, 200), "float32", "float32")
    y[:10] += 3000.0
    y[10:20] = 4.0
    y[20:30] = 0.0
    r[15:25] = 0.0
    gr, gn = make(torch, gen, 40, 200), make(torch, gen, 40, 200)
    for kind in ("layer", "rms"):
        check_norm(torch, ops, y, r, g, kw if kind == "layer" else {k: v for k, v in kw.items() if "bias" not in k}, gr, gn, kind=kind, act="sigmoid")


def test_block_norm_no_rows(env):
    torch, ops = env
    y = torch.empty((0, 64), device="cuda")
    w = torch.ones(64, device="cuda")
    assert ops.block_norm(y, y, y, scale=w)["normed"].shape == (0, 64)
    g = ops.block_norm_backward(y, y, y, grad_residual=y, grad_normed=y, scale=w, pre_weight=w)
    assert (g["grad_scale"] == 0).all() and (g["grad_pre_weight"] == 0).all()


# ------------------------------------------------------------------------------------------
# token_logprobs
# ------------------------------------------------------------------------------------------
def check_logprobs(torch, ops, z, tokens, n_top, gl, gh, ignore=-100):
    from oracle import sequence_ref as ref

    got = ops.token_logprobs(z, tokens, n_top=n_top, ignore_index=ignore, save=True)
    out = {k: v for k, v in got.items() if k != "stats" and v is not None}
    if gl is not None or gh is not None:
        out["grad_logits"] = ops.token_logprobs_backward(z, tokens, got["stats"], gl, gh, ignore_index=ignore)
    h = lambda t: None if t is None else host(t).reshape(-1)  # noqa: E731
    want, bound = ref.token_logprobs(host(z).reshape(-1, z.shape[-1]), None if tokens is None else tokens.cpu().numpy().reshape(-1), ignore, n_top, h(gl), h(gh))
    for name, t in out.items():
        if name == "top_ids":
            assert np.array_equal(t.cpu().numpy().reshape(want[name].shape), want[name]), "top_ids"
        else:
            check(name, t, want[name], bound[name])


def logit_inputs(torch, gen, rows, classes, dtype, token_dtype="int64", ignored=0.2, spread=3.0):
    z = make(torch, gen, rows, classes, dtype=dtype, scale=spread)
    t = torch.randint(0, classes, (rows,), generator=gen)
    if token_dtype != "uint8":
        t[torch.rand(rows, generator=gen) < ignored] = -100
    return z, t.to(getattr(torch, token_dtype)).cuda(), make(torch, gen, rows), make(torch, gen, rows)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,classes,n_top", [
    (1, 1, 1), (5, 2, 2), (1000, 2, 1), (77, 3, 3), (130, 5, 2), (64, 8, 8), (99, 9, 4), (333, 16, 0), (40, 17, 5), (65, 33, 32), (31, 64, 3), (9, 127, 1), (20, 255, 7),
    (6, 512, 32), (7, 513, 5), (5, 1000, 10), (3, 2048, 20), (4, 2049, 1), (3, 4096, 8), (2, 8191, 32), (1, 20000, 20), (2, 50257, 0)])
def test_token_logprobs_match_the_definition(env, dtype, rows, classes, n_top):
    torch, ops = env
    gen = torch.Generator().manual_seed(rows + classes)
    z, t, gl, gh = logit_inputs(torch, gen, rows, classes, dtype)
    check_logprobs(torch, ops, z, t, n_top, gl, gh)


@pytest.mark.parametrize("token_dtype", ["int8", "uint8", "int32", "int64"])
def test_token_logprobs_token_types(env, token_dtype):
    torch, ops = env
    gen = torch.Generator().manual_seed(31)
    for classes in (2, 16, 100):
        z, t, gl, gh = logit_inputs(torch, gen, 211, classes, "float32", token_dtype)
        check_logprobs(torch, ops, z, t, 2, gl, None)
        check_logprobs(torch, ops, z, t, 0, None, gh)


@pytest.mark.parametrize("classes", [2, 7, 64, 700, 3000])
def test_token_logprobs_forbidden_classes_and_empty_rows(env, classes):
    """-inf classes, rows of nothing else, a given token that is forbidden, the type's lowest value."""
    torch, ops = env
    gen = torch.Generator().manual_seed(32)
    z, t, gl, gh = logit_inputs(torch, gen, 60, classes, "float32")
    z[torch.rand(60, classes, generator=gen).cuda() < 0.4] = float("-inf")
    z[10:20] = float("-inf")
    z[20:30, 1:] = torch.finfo(torch.float32).min
    z[30:35, classes // 2:] = float("-inf")
    t[33] = classes - 1
    check_logprobs(torch, ops, z, t, min(4, classes), gl, gh)


@pytest.mark.parametrize("classes", [2, 50, 600, 5000])
def test_token_logprobs_nan_and_infinity(env, classes):
    """A NaN or +inf makes its own row NaN and no other; in a skipped row it is not read."""
    torch, ops = env
    gen = torch.Generator().manual_seed(33)
    z, t, gl, gh = logit_inputs(torch, gen, 40, classes, "bfloat16", ignored=0.0)
    z[3, classes - 1] = float("nan")
    z[5, 0] = float("inf")
    z[8] = float("nan")
    z[20:30] = float("nan")
    t[20:30] = -100
    check_logprobs(torch, ops, z, t, min(3, classes), gl, gh)


@pytest.mark.parametrize("classes", [2, 31, 513, 4097])
def test_token_logprobs_ties_go_to_the_lowest_class(env, classes):
    torch, ops = env
    gen = torch.Generator().manual_seed(34)
    z, t, gl, gh = logit_inputs(torch, gen, 30, classes, "float32")
    z = z.round()
    z[0] = 1.5
    z[1] = 0.0
    z[1, ::2] = -0.0
    check_logprobs(torch, ops, z, t, min(classes, 32), gl, gh)


def test_token_logprobs_confident_rows_keep_their_digits(env):
    """Two classes 5 to 80 apart: the winner's log probability is -exp(-gap), not 0."""
    torch, ops = env
    gap = torch.tensor([5.0, 12.0, 20.0, 40.0, 80.0])
    z = torch.stack([gap, torch.zeros(5)], 1).cuda()
    r = ops.token_logprobs(z, torch.zeros(5, dtype=torch.int8, device="cuda"))
    want = -torch.log1p(torch.exp(-gap.double()))
    assert ((r["logprob"].double().cpu() - want) / want).abs().max() < (2 * 80 + 8) * 2.0 ** -24


def test_token_logprobs_wrong_tokens(env):
    """A token outside the classes: NaN, nothing read out of the row."""
    torch, ops = env
    gen = torch.Generator().manual_seed(35)
    for classes in (2, 30, 900, 2500):
        z, t, gl, gh = logit_inputs(torch, gen, 20, classes, "float32", ignored=0.0)
        t[3], t[4], t[5], t[6] = -1, classes, 2 ** 40, -2 ** 60
        check_logprobs(torch, ops, z, t, 1, gl, gh)


@pytest.mark.parametrize("classes", [2, 16, 100, 777, 2300])
def test_token_logprobs_shapes_and_strides(env, classes):
    """[reads, length, classes] as the model returns it, rows that lie apart, unaligned rows, no tokens, no entropy."""
    torch, ops = env
    gen = torch.Generator().manual_seed(36)
    wide = make(torch, gen, 6, 11, classes + 5, dtype="bfloat16", scale=2.0)
    gl, gh = make(torch, gen, 6, 11), make(torch, gen, 6, 11)
    t = torch.randint(0, classes, (6, 11), generator=gen).cuda()
    for z in (wide[..., :classes], wide[..., 5:], wide[..., 3:3 + classes].contiguous()):
        check_logprobs(torch, ops, z, t, 2, gl, gh)
    check_logprobs(torch, ops, wide[..., 1:1 + classes], None, 1, None, gh)
    z = wide[..., :classes]
    assert ops.token_logprobs(z, t, want_entropy=False)["entropy"] is None
    one = z[:1, :1].expand(6, 11, classes)  # one row for all
    assert torch.equal(ops.token_logprobs(one, t, n_top=2)["top_ids"], ops.token_logprobs(one.contiguous(), t, n_top=2)["top_ids"])


def test_token_logprobs_no_rows(env):
    torch, ops = env
    z = torch.empty((0, 9), device="cuda")
    r = ops.token_logprobs(z, torch.empty(0, dtype=torch.int64, device="cuda"), n_top=3)
    assert r["logprob"].shape == (0,) and r["top_ids"].shape == (0, 3)
    assert ops.token_logprobs_backward(z, torch.empty(0, dtype=torch.int64, device="cuda"), None, r["logprob"]).shape == (0, 9)


def test_token_logprobs_rows_beyond_32_bits(env):
    """Rows 2^26 elements apart: the last start behind element 2^32."""
    torch, ops = env
    gen = torch.Generator().manual_seed(37)
    wide = torch.empty((70, 1 << 26), dtype=torch.bfloat16, device="cuda")
    z = wide[:, 5:905]
    z.copy_(torch.randn((70, 900), generator=gen))
    t = torch.randint(0, 900, (70,), generator=gen).cuda()
    gl, gh = make(torch, gen, 70), make(torch, gen, 70)
    check_logprobs(torch, ops, z, t, 3, gl, gh)


def test_token_logprobs_many_rows_of_a_wide_vocabulary(env):
    """More rows than one wave of workgroups, the last classes of the last row included."""
    torch, ops = env
    gen = torch.Generator().manual_seed(38)
    z = torch.randn((5000, 1111), device="cuda").bfloat16()
    t = torch.randint(0, 1111, (5000,), generator=gen).cuda()
    r = ops.token_logprobs(z, t, n_top=2, save=True)
    lp = torch.log_softmax(z.double(), -1)
    # 1 111 / 64 + 24 sums and 4 steps of the distance, as the oracle counts
    assert (r["logprob"].double() - lp.gather(1, t[:, None])[:, 0]).abs().max() < (1111 / 64 + 24 + 4 * 20) * 2.0 ** -24
    assert (r["entropy"].double() + (lp.exp() * lp).sum(-1)).abs().max() < (1111 / 64 + 24) * 22 * 2.0 ** -24
    assert (r["top_ids"][:, 0].long() == z.float().argmax(-1)).all() or (z.gather(1, r["top_ids"].long()[:, :1])[:, 0] == z.amax(-1)).all()


# ------------------------------------------------------------------------------------------
# streams, graphs, refusals
# ------------------------------------------------------------------------------------------
def layer_step(torch, ops, d):
    """One recurrent layer and its loss, forward and backward, through the three operators."""
    n = d["x"].shape[0]
    a = ops.block_norm(None, d["x"], pre_weight=d["w0"], pre_bias=d["b0"])
    proj = a["normed"] @ d["p"]
    c = d["x"].shape[1]
    x, f, gate = proj[:, :c], proj[:, c:2 * c], proj[:, 2 * c:]
    s = ops.gated_scan(x, f, offsets=d["off"], max_len=d["max_len"], h0=d["h0"], save=True, reverse=d["reverse"])
    kw = dict(kind="rms", gate_act="silu", scale=d["scale"], post_weight=d["w1"], pre_weight=d["w2"])
    b = ops.block_norm(s["y"], d["x"], gate, **kw)
    logits = b["normed"] @ d["e"]
    lp = ops.token_logprobs(logits, d["t"], n_top=2, save=True)
    gl = ops.token_logprobs_backward(logits, d["t"], lp["stats"], d["gl"], d["gh"])
    gb = ops.block_norm_backward(s["y"], d["x"], gate, grad_normed=gl @ d["et"], **kw)
    gs = ops.gated_scan_backward(x, f, s["saved"], gb["grad_y"], h0=d["h0"], offsets=d["off"], max_len=d["max_len"], reverse=d["reverse"])
    gp = torch.cat([gs["grad_x"], gs["grad_f"], gb["grad_gate"]], 1)
    ga = ops.block_norm_backward(None, d["x"], grad_residual=gb["grad_residual"], grad_normed=gp @ d["pt"], pre_weight=d["w0"], pre_bias=d["b0"])
    assert n == lp["logprob"].shape[0]
    return {"logprob": lp["logprob"], "entropy": lp["entropy"], "top": lp["top_ids"], "h": s["h_last"], "gx": ga["grad_residual"], "gw0": ga["grad_pre_weight"],
            "gb0": ga["grad_pre_bias"], "gw1": gb["grad_post_weight"], "gw2": gb["grad_pre_weight"], "gscale": gb["grad_scale"], "gh0": gs["grad_h0"]}


def layer_inputs(torch, seed, lengths, c, classes, reverse=False):
    gen = torch.Generator().manual_seed(seed)
    n = sum(lengths)
    d = {"x": make(torch, gen, n, c), "p": make(torch, gen, c, 3 * c, scale=c ** -0.5), "e": make(torch, gen, c, classes, scale=2 * c ** -0.5),
         "h0": make(torch, gen, len(lengths), c), "gl": make(torch, gen, n, scale=1 / n), "gh": make(torch, gen, n, scale=0.1 / n),
         "off": torch.tensor([0] + list(np.cumsum(lengths))).cuda(), "max_len": max(lengths), "reverse": reverse}
    for k in ("w0", "w1", "w2", "scale"):
        d[k] = make(torch, gen, c, scale=0.1, shift=1.0)
    d["b0"] = make(torch, gen, c, scale=0.1)
    t = torch.randint(0, classes, (n,), generator=gen)
    t[::9] = -100
    d["t"] = t.to(torch.int32).cuda()
    d["pt"], d["et"] = d["p"].t().contiguous(), d["e"].t().contiguous()
    return d


@pytest.mark.parametrize("reverse", [False, True])
def test_a_layer_of_all_three_against_autograd(env, reverse):
    """Norm, projection, recurrence, gated norm, logits and scores together, with every gradient, against torch's own differentiation in
    64 bits on the CPU.  Chained fp32 stages of unit-sized values: 1e-4 of each result's norm is 800 half steps."""
    torch, ops = env
    lengths, c, classes = [70, 1, 200, 33], 48, 700
    d = layer_inputs(torch, 41, lengths, c, classes, reverse)
    got = layer_step(torch, ops, d)
    q = {k: v.double().cpu() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in d.items()}
    leaves = {k: q[k].requires_grad_() for k in ("x", "w0", "b0", "w1", "w2", "scale", "h0")}
    proj = torch.nn.functional.layer_norm(q["x"], (c,), q["w0"], q["b0"], 1e-5) @ q["p"]
    xs, fs, gate = proj.split(c, 1)
    ys, hs = [None] * sum(lengths), []
    pos = 0
    for s, n in enumerate(lengths):
        h = q["h0"][s]
        for i in (range(pos + n - 1, pos - 1, -1) if reverse else range(pos, pos + n)):
            a = torch.sigmoid(fs[i])
            h = a * h + (1 - a) * xs[i]
            ys[i] = h
        hs.append(h)
        pos += n
    y = torch.stack(ys)
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt()  # noqa: E731
    r = q["x"] + q["scale"] * torch.nn.functional.silu(gate) * (rms(y) * q["w1"])
    logits = (rms(r) * q["w2"]) @ q["e"]
    lp = torch.log_softmax(logits, -1)
    t = d["t"].cpu().long()
    live = t != -100
    logprob = lp.gather(1, t.clamp_min(0)[:, None])[:, 0] * live
    entropy = -(lp.exp() * lp).sum(-1) * live
    ((logprob * q["gl"]).sum() + (entropy * q["gh"]).sum()).backward()
    want = {"logprob": logprob, "entropy": entropy, "h": torch.stack(hs), "gx": leaves["x"].grad, "gw0": leaves["w0"].grad, "gb0": leaves["b0"].grad,
            "gw1": leaves["w1"].grad, "gw2": leaves["w2"].grad, "gscale": leaves["scale"].grad, "gh0": leaves["h0"].grad}
    for k, w in want.items():
        off = (got[k].double().cpu() - w).norm() / w.norm()
        assert off < 1e-4, (k, float(off))


def test_side_stream_and_repeats_give_the_same_bits(env):
    torch, ops = env
    d = layer_inputs(torch, 42, [300, 5, 900], 64, 600)
    first = layer_step(torch, ops, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = layer_step(torch, ops, d)
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert torch.equal(first[k], second[k]), k


def test_graphs_replay_to_the_eager_results(env):
    """Two captured graphs of different sizes, replayed in turn with new inputs and eager work between: every replay is the eager result."""
    torch, ops = env
    sets = [layer_inputs(torch, 43, [40, 300], 64, 40), layer_inputs(torch, 44, [2500], 32, 1500)]
    graphs = []
    for d in sets:
        layer_step(torch, ops, d)  # (libraries make their handles outside the capture)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer_step(torch, ops, d)
        graphs.append((g, out))
    for turn in range(3):
        for d, (g, out) in zip(sets, graphs):
            d["x"].copy_(torch.randn(d["x"].shape, generator=torch.Generator().manual_seed(100 + turn)))
            g.replay()
            torch.cuda.synchronize()
            want = layer_step(torch, ops, d)
            for k in want:
                assert torch.equal(out[k], want[k]), (turn, k)


def test_wrappers_refuse(env):
    torch, ops = env
    from deepchopper_amd._lib import DeepChopperHipError

    z = torch.zeros((4, 8), device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    h = torch.zeros((1, 8), device="cuda")
    off = torch.tensor([0, 4]).cuda()
    for call in (lambda: ops.token_logprobs(z.cpu(), t), lambda: ops.token_logprobs(z, t.cpu()), lambda: ops.token_logprobs(z, t.float()),
                 lambda: ops.token_logprobs(z, t[:3]), lambda: ops.token_logprobs(z.double(), t), lambda: ops.token_logprobs(z.t(), t),
                 lambda: ops.token_logprobs(z[0], t[0]), lambda: ops.token_logprobs(z.view(2, 2, 8).transpose(0, 1), t.view(2, 2)),
                 lambda: ops.gated_scan(z, z), lambda: ops.gated_scan(z, z.half(), offsets=off), lambda: ops.gated_scan(z, z[:3], offsets=off),
                 lambda: ops.gated_scan(z, z, offsets=off.int()), lambda: ops.gated_scan(z, z, offsets=off, h0=h.half()),
                 lambda: ops.gated_scan(z, z, offsets=off, begin=off, end=off), lambda: ops.gated_scan(z, z, begin=off),
                 lambda: ops.gated_scan_backward(z, z, h, z, offsets=off, max_len=4, h0=h.t()), lambda: ops.gated_scan_backward(z, z, h[:0], z, offsets=off),
                 lambda: ops.block_norm(None, None), lambda: ops.block_norm(z, z, kind="batch"), lambda: ops.block_norm(z, z, z, gate_act="relu"),
                 lambda: ops.block_norm(z, z[:2]), lambda: ops.block_norm(z, z, z.half()), lambda: ops.block_norm(z, z, scale=h[0, :4]),
                 lambda: ops.block_norm(None, z, z)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.token_logprobs(z, t, n_top=9), lambda: ops.token_logprobs(torch.zeros((2, 99), device="cuda"), n_top=33),
                 lambda: ops.token_logprobs_backward(torch.zeros((4, 600), device="cuda"), t, None, torch.zeros(4, device="cuda")),
                 lambda: ops.token_logprobs_backward(z, None, None, torch.zeros(4, device="cuda")),
                 lambda: ops.gated_scan(z, z, offsets=off, out=z[:1].expand(4, 8)), lambda: ops.block_norm(z.half(), z.bfloat16()),
                 lambda: ops.block_norm(z, z, eps=-1.0), lambda: ops.block_norm(torch.zeros((1, 8193), device="cuda"))):
        with pytest.raises(DeepChopperHipError):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("padding", [False, True])
def test_predict_reads_scores(env, padding):
    """`predict_reads(want_scores=True)`: the log probability of every base's predicted label and the entropy, of the logits of that call."""
    torch, ops = env
    from deepchopper_amd import synth
    from deepchopper_amd.model import DeepChopper
    from deepchopper_amd.predict import PredictPipeline
    from deepchopper_amd.weights import synthetic_state_dict
    from oracle import sequence_ref as ref

    pipe = PredictPipeline(DeepChopper.from_state_dict(synthetic_state_dict(0)))
    rng = np.random.default_rng(45)
    reads = [synth.synth_reads_fixed(1, int(n), seed=int(n)) for n in rng.integers(30, 400, 5)]
    ids, seqs, quals = [f"r{i}" for i in range(5)], [r[0][0].tobytes() for r in reads], [r[1][0].tobytes() for r in reads]
    plain, _ = pipe.predict_reads(ids, seqs, quals, reference_padding=padding)
    out, res = pipe.predict_reads(ids, seqs, quals, reference_padding=padding, want_scores=True)
    logits = res["logits"].cpu().numpy()
    for i, (o, p) in enumerate(zip(out, plain)):
        assert "log_prob" not in p and o["intervals"] == p["intervals"] and np.array_equal(o["prediction"], p["prediction"])
        first, n = int(res["first"][i]), len(seqs[i])
        want, bound = ref.token_logprobs(logits[i, first:first + n], n_top=1)
        assert o["log_prob"].shape == o["entropy"].shape == (n,) and np.array_equal(want["top_ids"][:, 0], o["prediction"])
        for name, w, b in (("log_prob", want["top_logprob"][:, 0], bound["top_logprob"][:, 0]), ("entropy", want["entropy"], bound["entropy"])):
            assert (np.abs(o[name] - w) <= b + HALF_STEP["float32"] * np.abs(w) + TINY["float32"]).all(), name


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,c", [("float32", 5), ("bfloat16", 131), ("float16", 64)])
def test_gated_scan_short_sequences_at_begin_and_end(env, reverse, dtype, c):
    """Up to 16 tokens of each row, gaps and sequences that break the contract among them: the token-by-token form."""
    torch, ops = env
    from oracle import sequence_ref as ref

    gen = torch.Generator().manual_seed(46)
    n = 120
    x, f, gy = (make(torch, gen, n, c, dtype=dtype) for _ in range(3))
    ranges = [(100, 112), (3, 3), (7, 8), (20, 36), (60, 59), (110, 121), (40, 57)]
    good = [0, 1, 2, 3]
    b, e = (torch.tensor([r[i] for r in ranges]).cuda() for i in (0, 1))
    r = ops.gated_scan(x, f, begin=b, end=e, max_len=16, reverse=reverse, save=True)
    g = ops.gated_scan_backward(x, f, r["saved"], gy, begin=b, end=e, max_len=16, reverse=reverse)
    want, bound = ref.gated_scan(host(x), host(f), [ranges[i] for i in good], None, reverse, host(gy))
    covered = torch.from_numpy(~np.isnan(want["y"][:, 0])).cuda()
    for name, t in {"y": r["y"], "grad_x": g["grad_x"], "grad_f": g["grad_f"]}.items():
        check(name, t[covered], want[name][covered.cpu().numpy()], bound[name][covered.cpu().numpy()])
        assert (t[~covered] == 0).all()
    for name, t in {"h_last": r["h_last"], "grad_h0": g["grad_h0"]}.items():
        check(name, t[good], want[name], bound[name])
        assert torch.isnan(t[4:]).all()


def test_gated_scan_of_padded_rows_in_a_graph(env):
    """begin / end inside a captured graph: the gaps are cleared at every replay."""
    torch, ops = env
    gen = torch.Generator().manual_seed(47)
    x, f = make(torch, gen, 300, 32), make(torch, gen, 300, 32)
    b, e = torch.tensor([10, 150]).cuda(), torch.tensor([90, 300]).cuda()
    ops.gated_scan(x, f, begin=b, end=e, max_len=150)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.gated_scan(x, f, begin=b, end=e, max_len=150)
    for turn in range(4):
        x.copy_(torch.randn((300, 32), generator=gen))
        b.copy_(torch.tensor([10 + turn, 150 + turn]))
        out["y"].fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        want = ops.gated_scan(x, f, begin=b, end=e, max_len=150)
        assert torch.equal(out["y"], want["y"]) and torch.equal(out["h_last"], want["h_last"]), turn


def test_block_norm_first_norm_in_another_type(env):
    """The first norm of a model: an fp32 stream in, 16-bit activations out, and back."""
    torch, ops = env
    from oracle import sequence_ref as ref

    gen = torch.Generator().manual_seed(48)
    for w in (64, 300):
        r, gr, gn = make(torch, gen, 40, w), make(torch, gen, 40, w), make(torch, gen, 40, w, dtype="bfloat16")
        q = make(torch, gen, w, shift=1.0, scale=0.1)
        got = ops.block_norm(None, r, pre_weight=q, dtype=torch.bfloat16)
        back = ops.block_norm_backward(None, r, grad_residual=gr, grad_normed=gn, pre_weight=q)
        want, bound = ref.block_norm(None, host(r), None, kind="layer", act="identity", pre_weight=host(q), grad_residual=host(gr), grad_normed=host(gn))
        assert got["normed"].dtype == torch.bfloat16 and back["grad_residual"].dtype == torch.float32
        check("normed", got["normed"], want["normed"], bound["normed"])
        for k in ("grad_residual", "grad_pre_weight"):
            check(k, back[k], want[k], bound[k])


@pytest.mark.parametrize("classes", [2, 40, 300, 513, 9001])
def test_token_logprobs_gradient_in_place_of_the_logits(env, classes):
    """The C entry takes d_logits as d_grad_logits."""
    torch, ops = env
    from deepchopper_amd import _lib

    gen = torch.Generator().manual_seed(49)
    z, t, gl, gh = logit_inputs(torch, gen, 33, classes, "float16")
    r = ops.token_logprobs(z, t, save=True)
    want = ops.token_logprobs_backward(z, t, r["stats"], gl, gh)
    _lib.check(_lib.lib().dc_token_logprobs_backward(torch.cuda.current_stream().cuda_stream, z.data_ptr(), 1, 33, classes, classes, t.data_ptr(), 3, -100,
                                                     None if r["stats"] is None else r["stats"].data_ptr(), gl.data_ptr(), gh.data_ptr(), z.data_ptr(), classes))
    assert torch.equal(z, want)
