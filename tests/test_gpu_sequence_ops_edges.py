"""GPU tests of the sequence-layer and scoring operators where a call leaves the ordinary: refused sequences, values at the end of
fp32's range, gates that are all but open, sure predictions, arguments that are not used."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env(hip_lib):
    import torch

    from deepchopper_amd import _lib, ops

    assert _lib.device_count() >= 1, "GPU tests need a HIP device; there is no CPU fallback"
    return torch, ops


HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}  # half the smallest step (fp32 results below 2^-126 may be flushed)


def check(name, got, want, bound):
    """Off by no more than the bound for 32 bits and half a step of the output's type; what is not finite has to be the same."""
    dt = str(got.dtype).replace("torch.", "")
    g = host(got).reshape(want.shape)
    with np.errstate(invalid="ignore"):
        off = np.abs(g - want) - (bound + HALF_STEP[dt] * (np.abs(want) + bound) + TINY[dt])
        right = np.where(np.isfinite(want), off <= 0, (g == want) | (np.isnan(g) & np.isnan(want)))
    assert right.all(), f"{name}: {(~right).sum()} of {want.size} values off, first at {tuple(np.argwhere(~right)[0])}: {g[~right][:4]} for {want[~right][:4]}"


def host(t):
    return t.detach().double().cpu().numpy()


def randn(torch, gen, *shape, dtype="float32", scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen) * scale + shift).to(getattr(torch, dtype)).cuda()


# ------------------------------------------------------------------------------------------
# gated_scan: sequences that are refused
# ------------------------------------------------------------------------------------------
def poison(torch, *tensors):
    """Blocks of these tensors' sizes, full of 77, go back to the allocator: what a call does not write shows as 77."""
    blocks = [torch.full_like(t, 77.0) for t in tensors for _ in range(4)]
    torch.cuda.synchronize()
    del blocks


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,c", [("float32", 40), ("bfloat16", 33), ("float16", 130)])
@pytest.mark.parametrize("offsets,max_len,refused", [
    ([0, 50, 120, 400], 200, [2]),           # longer than the bound
    ([20, 30, 46, 60, 400], 16, [3]),        # ... in the token-by-token form
    ([0, 50, 4000, 5000], 5000, [1, 2]),     # past the tokens, in part and altogether; chunked
    ([-30, 40, 90, 400], 400, [0]),          # in front of them
    ([-8, 4, 9, 25], 16, [0]),
])
def test_gated_scan_rows_of_a_refused_sequence_are_nan(env, reverse, dtype, c, offsets, max_len, refused):
    torch, ops = env
    gen = torch.Generator().manual_seed(51)
    n, k = 420, len(offsets) - 1
    x, f, gy = (randn(torch, gen, n, c, dtype=dtype) for _ in range(3))
    h0 = randn(torch, gen, k, c)
    off = torch.tensor(offsets).cuda()
    kw = dict(offsets=off, max_len=max_len, h0=h0, reverse=reverse)
    poison(torch, x)
    r = ops.gated_scan(x, f, save=True, **kw)
    poison(torch, x)
    g = ops.gated_scan_backward(x, f, r["saved"], gy, grad_h_last=h0, **kw)
    for s in range(k):
        b, e = (min(max(offsets[s + i], 0), n) for i in (0, 1))
        for t in (r["y"], g["grad_x"], g["grad_f"]):
            assert torch.isnan(t[b:e]).all() if s in refused else not torch.isnan(t[b:e]).any(), s
        for t in (r["h_last"], g["grad_h0"]):
            assert torch.isnan(t[s]).all() if s in refused else not torch.isnan(t[s]).any(), s
        if s not in refused:  # the others: as if they were alone
            one = dict(offsets=torch.tensor([0, e - b]).cuda(), max_len=e - b, h0=h0[s:s + 1].contiguous(), reverse=reverse)
            xs, fs, gs = (t[b:e].contiguous() for t in (x, f, gy))
            alone = ops.gated_scan(xs, fs, save=True, **one)
            back = ops.gated_scan_backward(xs, fs, alone["saved"], gs, grad_h_last=h0[s:s + 1].contiguous(), **one)
            for t, w in ((r["y"], alone["y"]), (g["grad_x"], back["grad_x"]), (g["grad_f"], back["grad_f"])):
                assert torch.allclose(t[b:e].float(), w.float(), rtol=2.0 ** -7, atol=1e-4)  # (divided otherwise, so not the same bits: a step of 16 bits, or fp32 noise)
    first, last = (min(max(o, 0), n) for o in (offsets[0], offsets[-1]))
    for t in (r["y"], g["grad_x"], g["grad_f"]):
        assert (t[:first] == 0).all() and (t[last:] == 0).all()


def test_gated_scan_one_refused_sequence_among_many(env):
    """More sequences than a wavefront looks at in one go."""
    torch, ops = env
    gen = torch.Generator().manual_seed(52)
    lens = [2] * 20000
    for s in (0, 63, 64, 9999, 19999):
        lens[s] = 6
    off = torch.tensor([0] + lens).cumsum(0)
    n, c = int(off[-1]), 6
    x, f = randn(torch, gen, n, c), randn(torch, gen, n, c)
    for max_len in (5, 6):
        poison(torch, x)
        r = ops.gated_scan(x, f, offsets=off.cuda(), max_len=max_len)
        bad = torch.tensor(lens) > max_len
        assert torch.equal(torch.isnan(r["h_last"]).all(1).cpu(), bad)
        assert torch.equal(torch.isnan(r["y"]).all(1).cpu(), bad.repeat_interleave(torch.tensor(lens)))


def test_gated_scan_refused_sequences_leave_a_given_out(env):
    """`out` of the caller's: rows of a refused sequence are nobody's to write."""
    torch, ops = env
    gen = torch.Generator().manual_seed(53)
    x, f = randn(torch, gen, 100, 8), randn(torch, gen, 100, 8)
    out = torch.full((100, 8), 5.0, device="cuda")
    r = ops.gated_scan(x, f, offsets=torch.tensor([10, 30, 90]).cuda(), max_len=20, out=out)
    assert (out[:10] == 5).all() and (out[30:] == 5).all() and (out[10:30] != 5).any(1).all() and torch.isnan(r["h_last"][1]).all()


# ------------------------------------------------------------------------------------------
# gated_scan: the end of fp32's range
# ------------------------------------------------------------------------------------------
def scan_against_the_definition(torch, ops, x, f, lengths, h0, gy, gl, reverse):
    from oracle import sequence_ref as ref

    ends = np.cumsum(lengths)
    kw = dict(offsets=torch.tensor([0] + list(ends)).cuda(), max_len=max(lengths), h0=h0, reverse=reverse)
    got = ops.gated_scan(x, f, save=True, **kw)
    got.update(ops.gated_scan_backward(x, f, got["saved"], gy, grad_h_last=gl, **kw))
    with np.errstate(invalid="ignore"):
        want, bound = ref.gated_scan(host(x), host(f), [(int(e - n), int(e)) for e, n in zip(ends, lengths)], host(h0), reverse, host(gy), host(gl))
    for name in want:
        check(name, got[name], want[name], bound[name])
    return got, want


# token by token; tiles; whole tiles; chunks of one and of two channels a lane; narrow rows
SIZES = [([7, 16, 1, 0], 33), ([300, 17, 0], 48), ([1000, 130], 128), ([9001, 0, 700], 64), ([5000], 130), ([3000, 40], 5)]


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths,c", SIZES)
def test_gated_scan_of_the_largest_numbers(env, lengths, c, dtype, reverse):
    """States between inputs of the type's largest and lowest values are finite: x - h is not.  (Gradients of 0.02, so that theirs are too.)"""
    torch, ops = env
    gen = torch.Generator().manual_seed(54)
    n, k, most = sum(lengths), len(lengths), torch.finfo(getattr(torch, dtype)).max

    def huge(*shape):
        t = torch.rand(shape, generator=gen) * 0.5 + 0.5
        t[torch.rand(shape, generator=gen) < 0.3] = 1.0
        return t * torch.where(torch.rand(shape, generator=gen) < 0.5, -most, most)

    x, h0 = huge(n, c).to(getattr(torch, dtype)).cuda(), huge(k, c).cuda()
    x[: n // 3, 0] = -most  # a column that stays at the lowest value for long
    f = randn(torch, gen, n, c, dtype=dtype, scale=2.0)
    f[:, -1] += 5.0  # ... and one of a long memory
    gy, gl = randn(torch, gen, n, c, dtype=dtype, scale=0.005), randn(torch, gen, k, c, scale=0.02)
    got, want = scan_against_the_definition(torch, ops, x, f, lengths, h0, gy, gl, reverse)
    assert np.isfinite(want["y"]).all() and torch.isfinite(got["y"]).all()


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("lengths,c", SIZES)
def test_gated_scan_infinities_go_as_the_definition_says(env, lengths, c, dtype, reverse):
    """An infinite input or state, or one of either sign and then NaN, from there on; infinite gradients; other channels as ever."""
    torch, ops = env
    gen = torch.Generator().manual_seed(55)
    n, k = sum(lengths), len(lengths)
    x, f, gy = (randn(torch, gen, n, c, dtype=dtype) for _ in range(3))
    h0, gl = randn(torch, gen, k, c), randn(torch, gen, k, c)
    x[n // 2, 0] = float("inf")
    x[n // 3, 1] = float("-inf")
    x[2 * n // 3, 1] = float("inf")
    h0[:, 2] = float("inf")
    gy[n // 2, 3] = float("-inf")
    gl[:, 4] = float("inf")
    x[n // 4, c - 1] = float("nan")
    f[:, 0] -= 6.0  # strongly forgetting
    f[:, 2] += 20.0  # keeping: weights below fp32's last digit
    scan_against_the_definition(torch, ops, x, f, lengths, h0, gy, gl, reverse)


# ------------------------------------------------------------------------------------------
# gated_scan: every form against the definition
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,lengths,c", [
    ("float32", [9001], 64), ("bfloat16", [9001], 128), ("float16", [9001], 129), ("bfloat16", [4500, 17], 256),  # chunks of whole tiles
    ("float32", [1000] * 20, 192), ("bfloat16", [200, 64, 900], 512), ("float16", [130, 700], 768)])              # more than one block of full lanes
def test_gated_scan_whole_tiles_and_blocks_of_channels(env, dtype, lengths, c, reverse):
    torch, ops = env
    gen = torch.Generator().manual_seed(60)
    n, k = sum(lengths), len(lengths)
    x, f, gy = (randn(torch, gen, n, c, dtype=dtype) for _ in range(3))
    f = (f.float() * 2 + 3).to(f.dtype)
    scan_against_the_definition(torch, ops, x, f, lengths, randn(torch, gen, k, c), gy, randn(torch, gen, k, c), reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,c", [("float32", 64), ("bfloat16", 50), ("float16", 33), ("float32", 6)])
def test_gated_scan_in_chunks_with_gaps_empty_and_refused_sequences(env, dtype, c, reverse):
    """begin / end of long, short, empty and refused sequences, divided into chunks, with states and gradients of states."""
    torch, ops = env
    from oracle import sequence_ref as ref

    gen = torch.Generator().manual_seed(61)
    n, max_len = 9000, 5000
    ranges = [(3000, 8000), (100, 130), (1000, 1000), (-4, 30), (150, 900), (2000, 8900), (8500, 9001), (40, 39), (8999, 9000), (0, 0)]
    good = [i for i, (b, e) in enumerate(ranges) if 0 <= b <= e <= n and e - b <= max_len]
    bad = [i for i in range(len(ranges)) if i not in good]
    assert ops._lib.lib().dc_gated_scan_workspace(n, c, len(ranges), max_len) > 0  # (chunks have maps)
    x, f, gy = (randn(torch, gen, n, c, dtype=dtype) for _ in range(3))
    f = (f.float() * 2 + 2).to(f.dtype)
    h0, gl = randn(torch, gen, len(ranges), c), randn(torch, gen, len(ranges), c)
    b, e = (torch.tensor([r[i] for r in ranges]).cuda() for i in (0, 1))
    kw = dict(begin=b, end=e, max_len=max_len, h0=h0, reverse=reverse)
    r = ops.gated_scan(x, f, save=True, **kw)
    g = ops.gated_scan_backward(x, f, r["saved"], gy, grad_h_last=gl, **kw)
    want, bound = ref.gated_scan(host(x), host(f), [ranges[i] for i in good], host(h0)[good], reverse, host(gy), host(gl)[good])
    covered = ~np.isnan(want["y"][:, 0])
    inside = torch.from_numpy(covered).cuda()
    for name, t in (("y", r["y"]), ("grad_x", g["grad_x"]), ("grad_f", g["grad_f"])):
        check(name, t[inside], want[name][covered], bound[name][covered])
        assert (t[~inside] == 0).all()
    for name, t in (("h_last", r["h_last"]), ("grad_h0", g["grad_h0"])):
        check(name, t[good], want[name], bound[name])
        assert torch.isnan(t[bad]).all()
    out = torch.full((n, c), 5.0, device="cuda").to(x.dtype)
    again = ops.gated_scan(x, f, out=out, **kw)
    assert (out[~inside] == 5).all() and torch.equal(out[inside], r["y"][inside]) and torch.equal(again["h_last"][good], r["h_last"][good])


# ------------------------------------------------------------------------------------------
# block_norm
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", [8, 64, 250, 600])
def test_block_norm_slope_of_gates_that_are_all_but_open(env, width, dtype, act):
    """r' = act(gate) alone: its gradient is s (1 - s), or s (1 + x (1 - s)), with relative accuracy also where s rounds to 1.

    exp(-x) by a rounded x log2(e) (1.5 |x| half steps) and a one-ulp exp2 (2), 1 + e and a one-ulp reciprocal (3), e s (1), the product of
    the two (1), each error but the last ones in both factors: (1.5 |x| + 12) half steps; silu's x (1 - s) has another 1.5 |x|."""
    torch, ops = env
    from oracle.sequence_ref import U

    rows = 40
    x = torch.linspace(-80.0, 80.0, rows * width).reshape(rows, width)
    x[0] = torch.linspace(-30.0, 30.0, width)
    x[1, :6] = torch.tensor([12.0, 15.0, 17.0, 30.0, -12.0, 0.0])
    x[2, :2] = torch.tensor([float("inf"), torch.finfo(torch.float32).min / 2])
    gate = x.to(getattr(torch, dtype)).cuda()
    one = torch.ones((rows, width), dtype=gate.dtype, device="cuda")
    if act == "silu":
        gate[2, 0] = 80.0  # (x (1 - s) of an infinite x is no number)
    got = ops.block_norm_backward(one, None, gate, post=False, gate_act=act, grad_residual=one)["grad_gate"]
    x = host(gate)
    with np.errstate(over="ignore", invalid="ignore"):
        s, rest = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
        want = s * rest if act == "sigmoid" else s * (1 + x * rest)
        bound = (1.5 * np.abs(x) + 12) * U * np.abs(want) if act == "sigmoid" else (3 * np.abs(x) + 14) * U * s * (1 + np.abs(x) * rest)
    bound = np.where(np.isfinite(x), np.minimum(bound, 1.0), 0.0)  # (beyond 88 the slope is below fp32's normal numbers)
    check("grad_gate", got, want, bound)


@pytest.mark.parametrize("width", [64, 600])
@pytest.mark.parametrize("with_y,post,with_normed", [(True, 0, True), (True, 1, False), (False, 1, True), (True, 0, False)])
def test_block_norm_gradients_of_vectors_that_were_not_used_are_zero(env, width, with_y, post, with_normed):
    """The C entry with all five vectors' pointers: without a norm behind the block, without the next block's, without a block."""
    torch, ops = env
    from deepchopper_amd import _lib

    gen = torch.Generator().manual_seed(57)
    rows = 70
    y, r, gr, gn = (randn(torch, gen, rows, width) for _ in range(4))
    w = [randn(torch, gen, width, shift=1.0) for _ in range(4)]
    out = [torch.full((width,), 77.0, device="cuda") for _ in range(5)]
    grads = [torch.empty((rows, width), device="cuda") for _ in range(2)]
    L = _lib.lib()
    nb = L.dc_block_norm_workspace(rows, width, 0)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    at = lambda t, used=True: t.data_ptr() if used else None  # noqa: E731
    _lib.check(L.dc_block_norm_backward(torch.cuda.current_stream().cuda_stream, 0, 0, rows, width, 0, 1e-5, at(y, with_y), width, None, 0, 0, at(r), width,
                                        at(w[0]), post, at(w[1]), at(w[2]), at(w[3]), at(gr), width, at(gn, with_normed), width, at(grads[0], with_y), None,
                                        at(grads[1]), *(t.data_ptr() for t in out), ws.data_ptr(), nb))
    for t, used in zip(out, (with_y, with_y and post, with_y and post, with_normed, with_normed)):
        assert (t != 0).any() and (t != 77).all() if used else (t == 0).all()


# ------------------------------------------------------------------------------------------
# token_logprobs
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("classes", [2, 3, 4, 5, 16, 50, 100, 300, 512])
def test_token_logprobs_gradient_of_a_sure_row_keeps_its_digits(env, classes, dtype):
    """A given class 5 to 70 above the others: its gradient is g (1 - p), not 0, and a row's gradients add up to 0.

    log p keeps its digits to (2 gap + 8) half steps as a log1p of a sum (of up to 16 terms a lane and 5 steps over lanes: 21 more), the
    series of 1 - p to 8 and the product to 1.  Classes a little above give the other form of 1 - p: p is off by (2 |log p| + 4) half steps
    besides log p's 30, and at least a fifth of 1 is left: 5 times that."""
    torch, ops = env
    from oracle.sequence_ref import U

    gen = torch.Generator().manual_seed(56)
    gaps = torch.tensor([70.0, 60.0, 40.0, 25.0, 16.0, 9.0, 5.0, 3.0, 2.0, 1.0, 0.5])
    z = torch.rand((len(gaps), classes), generator=gen) * -2 - gaps[:, None] - np.log(classes)
    t = torch.randint(0, classes, (len(gaps),), generator=gen)
    z[torch.arange(len(gaps)), t] = 0.0
    z = z.to(getattr(torch, dtype)).cuda()
    g = torch.linspace(0.5, 2.0, len(gaps))
    got = ops.token_logprobs_backward(z, t.cuda(), None, g.cuda())
    zd, rows = host(z), np.arange(len(gaps))
    e = np.exp(zd)
    others = e.sum(1) - 1 if classes < 2 else np.array([np.delete(e[i], int(t[i])).sum() for i in rows])
    want = g.double().numpy() * others / (1 + others)
    gap = -np.sort(zd, 1)[:, -2]
    bound = np.where(others < 0.25, 2 * gap + 40, 5 * 40) * U * want
    check("given", got[torch.arange(len(gaps)), t.cuda()], want, bound)
    if dtype == "float32":
        total = host(got).sum(1)  # the other classes' gradients -g p_j are as accurate, and each is rounded once
        assert (np.abs(total) <= 2 * (bound + (2 * (gap + 2 + np.log(classes)) + 40) * U * want)).all()


# ------------------------------------------------------------------------------------------
# outputs that the caller gives
# ------------------------------------------------------------------------------------------
def test_given_outputs_that_share_elements_with_an_input_are_refused(env):
    torch, ops = env
    gen = torch.Generator().manual_seed(58)
    n, c = 200, 16
    wide = randn(torch, gen, n + 1, 3 * c)
    x, f, free = wide[:n, :c], wide[:n, c:2 * c], wide[:n, 2 * c:]
    off = torch.tensor([0, n]).cuda()
    kw = dict(offsets=off, max_len=n)
    want = ops.gated_scan(x, f, **kw)["y"]
    for out in (x, f, wide[1:, :c], wide[:n, 1:c + 1], wide[:n, 2 * c - 1:-1], wide[1:, 2 * c - 3:-3], wide.view(-1)[5:5 + n * c].view(n, c)):
        kept = wide.clone()
        with pytest.raises(ValueError, match="shares elements"):
            ops.gated_scan(x, f, out=out, **kw)
        assert torch.equal(wide, kept)
    # other columns, other rows, a row that is repeated: apart
    assert torch.equal(ops.gated_scan(x, f, out=free, **kw)["y"], want)
    some = dict(offsets=torch.tensor([0, 50]).cuda(), max_len=50)
    assert torch.equal(ops.gated_scan(x[:50], f[:50], out=wide[100:150, :c], **some)["y"], want[:50])
    every = torch.empty((100, 2, c), device="cuda")  # every other row
    every[:, 0] = x[:100]
    ops.gated_scan(every[:, 0], f[:100], out=every[:, 1], offsets=torch.tensor([0, 100]).cuda(), max_len=100)
    assert torch.equal(every[:, 1], ops.gated_scan(x[:100], f[:100], offsets=torch.tensor([0, 100]).cuda(), max_len=100)["y"])
    h = torch.zeros(2 * c, device="cuda")
    with pytest.raises(ValueError, match="h_last: shares elements with h0"):
        ops.gated_scan(x, f, h0=h[:c].view(1, c), h_last=h[1:c + 1].view(1, c), **kw)
    ops.gated_scan(x, f, h0=h[:c].view(1, c), h_last=h[c:].view(1, c), **kw)


@pytest.mark.parametrize("width", [24, 256, 700])
def test_block_norm_in_place_of_an_input(env, width):
    """r' in the place of the residual, the block's output or the gate, row for row; shifted by a row or a column it is refused."""
    torch, ops = env
    gen = torch.Generator().manual_seed(59)
    rows = 3000
    y, r, g = (randn(torch, gen, rows + 1, width + 4)[:, :width] for _ in range(3))
    want = ops.block_norm(y[:rows], r[:rows], g[:rows])
    for k in range(3):
        a = [t.clone() for t in (y, r, g)]
        a[k] = torch.empty((rows + 1, width + 4), device="cuda")[:, :width].copy_(a[k])
        got = ops.block_norm(*(t[:rows] for t in a), out=a[k][:rows])
        assert torch.equal(got["residual"], want["residual"]) and torch.equal(got["normed"], want["normed"])
        with pytest.raises(ValueError, match="shares elements"):
            ops.block_norm(*(t[:rows] for t in a), out=a[k][1:])
    with pytest.raises(ValueError, match="shares elements"):
        ops.block_norm(y[:rows].bfloat16(), r[:rows], out=r.as_strided((rows, width), (width + 4, 1), 1))
