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
