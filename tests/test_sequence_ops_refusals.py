"""CPU tests: what the C entry points of the sequence-layer and scoring operators refuse before anything is launched, their size functions,
and that calls with nothing to do need no GPU."""
import ctypes as C

import pytest

INVALID = 1
P = C.c_void_p(4096)  # a pointer that is looked at but never followed
ODD = C.c_void_p(4097)


@pytest.fixture(scope="module")
def L(hip_lib):
    from deepchopper_amd import _lib

    return _lib.lib()


def refused(L, rc, text):
    assert rc == INVALID and text in L.dc_last_error().decode(), (rc, L.dc_last_error())


def logprobs(L, z=P, dtype=0, n=4, classes=8, stride=8, tok=P, ttype=3, top=0, ids=None, top_lp=None):
    return L.dc_token_logprobs(None, z, dtype, n, classes, stride, tok, ttype, -100, top, P, P, None, ids, top_lp, None, 0)


def test_token_logprobs_refusals(L):
    refused(L, logprobs(L, z=None), "null pointer")
    refused(L, logprobs(L, dtype=3), "element type")
    refused(L, logprobs(L, ttype=4), "token type")
    refused(L, logprobs(L, n=-1), "negative size")
    refused(L, logprobs(L, classes=0), "negative size")
    refused(L, logprobs(L, classes=(1 << 30) + 1, stride=1 << 31), "2^30")
    refused(L, logprobs(L, stride=-8), "negative stride")
    refused(L, logprobs(L, z=ODD, dtype=1), "misaligned")
    refused(L, logprobs(L, tok=ODD), "misaligned")
    refused(L, logprobs(L, top=9, ids=P, top_lp=P), "n_top")
    refused(L, logprobs(L, classes=100, stride=100, top=33, ids=P, top_lp=P), "n_top")
    refused(L, logprobs(L, top=2, ids=P), "null pointer")
    back = lambda z=P, classes=8, tok=P, stats=None, gl=P, out=P, ld=8: L.dc_token_logprobs_backward(  # noqa: E731
        None, z, 0, 4, classes, classes, tok, 3, -100, stats, gl, None, out, ld)
    refused(L, back(out=None), "null pointer")
    refused(L, back(tok=None), "without tokens")
    refused(L, back(classes=513, ld=513), "statistics")
    refused(L, back(ld=7), "overlap")
    refused(L, back(out=ODD), "misaligned")
    assert logprobs(L, z=None, n=0) == 0


def scan(L, x=P, f=P, dtype=0, xs=8, n=100, c=8, b=P, e=P, seqs=2, longest=50, y=P, ys=8, ws=None, nb=0):
    return L.dc_gated_scan(None, dtype, x, xs, f, 8, n, c, b, e, seqs, longest, 0, None, y, ys, 0, None, None, ws, nb)


def test_gated_scan_refusals(L):
    refused(L, scan(L, x=None), "null pointer")
    refused(L, scan(L, y=None), "null pointer")
    refused(L, scan(L, dtype=-1), "element type")
    refused(L, scan(L, c=0), "size")
    refused(L, scan(L, n=-1), "size")
    refused(L, scan(L, longest=-1), "size")
    refused(L, scan(L, e=None), "come together")
    refused(L, scan(L, b=None, e=None, seqs=3), "exceed")
    refused(L, scan(L, xs=-1), "negative stride")
    refused(L, scan(L, ys=7), "overlap")
    refused(L, scan(L, x=ODD), "misaligned")
    refused(L, scan(L, seqs=1 << 30, c=256), "2^20")
    back = lambda saved=P, gy=P, gx=P, gxs=8, gf=P: L.dc_gated_scan_backward(  # noqa: E731
        None, 0, P, 8, P, 8, 100, 8, P, P, 2, 50, 0, None, saved, gy, 8, None, gx, gxs, gf, 8, 0, None, P, 1 << 30)
    refused(L, back(saved=None), "null pointer")
    refused(L, back(gy=None), "null pointer")
    refused(L, back(gf=None), "null pointer")
    refused(L, back(gxs=5), "overlap")
    refused(L, back(gx=ODD), "misaligned")
    # nothing to do, whatever the longest sequence might be
    assert scan(L, seqs=0, longest=100000) == 0 and scan(L, seqs=0, n=0, x=None, f=None, y=None, longest=100000) == 0
    assert L.dc_gated_scan_workspace(100, 8, 0, 100000) == 0 and L.dc_gated_scan_workspace(0, 8, 3, 100000) == 0
    # one long sequence needs the maps of its chunks, 16 tokens a step at a time nothing
    assert L.dc_gated_scan_workspace(100000, 64, 1, 100000) > 0 and L.dc_gated_scan_workspace(1600, 64, 100, 16) == 0
    refused(L, scan(L, n=100000, c=8, seqs=1, longest=100000), "workspace")
    # a bound on the lengths is no more than the tokens, however large
    assert L.dc_gated_scan_workspace(5000, 64, 2, 1 << 62) == L.dc_gated_scan_workspace(5000, 64, 2, 5000)
    assert L.dc_gated_scan_saved(0, 8) == 0 and L.dc_gated_scan_saved(1, 8) == 8 and L.dc_gated_scan_saved(65, 8) == 16
    assert L.dc_gated_scan_saved(1 << 33, 256) == 1 << 35


def norm(L, dtype=0, rdtype=0, n=4, w=8, kind=0, eps=1e-5, y=P, g=P, act=1, r=P, out=P, outs=8, normed=P):
    return L.dc_block_norm(None, dtype, rdtype, n, w, kind, eps, y, 8, g, 8, act, r, 8, None, 1, None, None, None, None, out, outs, normed, 8)


def test_block_norm_refusals(L):
    refused(L, norm(L, dtype=5), "element type")
    refused(L, norm(L, dtype=1, rdtype=2), "residual stream")
    refused(L, norm(L, rdtype=1), "residual stream")
    refused(L, norm(L, n=-1), "negative size")
    refused(L, norm(L, w=0), "width")
    refused(L, norm(L, w=8193), "width")
    refused(L, norm(L, kind=2), "unknown norm")
    refused(L, norm(L, act=3), "activation")
    refused(L, norm(L, eps=-1.0), "eps")
    refused(L, norm(L, eps=float("nan")), "eps")
    refused(L, norm(L, eps=float("inf")), "eps")
    refused(L, norm(L, y=None, g=None, r=None), "neither")
    refused(L, norm(L, y=None), "gate without")
    refused(L, norm(L, outs=4), "overlap")
    refused(L, norm(L, normed=ODD), "misaligned")
    back = lambda ws=P, nb=1 << 30, n=4: L.dc_block_norm_backward(  # noqa: E731
        None, 0, 0, n, 8, 0, 1e-5, P, 8, None, 0, 0, P, 8, None, 1, None, None, None, P, 8, P, 8, P, None, P, None, None, None, None, None, ws, nb)
    refused(L, back(ws=None), "workspace")
    refused(L, back(nb=L.dc_block_norm_workspace(4, 8, 0) - 1), "workspace")
    refused(L, back(ws=C.c_void_p(4100)), "workspace")
    assert L.dc_block_norm_workspace(0, 8, 0) == 0 and L.dc_block_norm_workspace(1 << 40, 8192, 2) < 1 << 31
    assert norm(L, n=0) == 0 and norm(L, out=None, normed=None) == 0


def test_wrappers_refuse_host_tensors():
    import torch

    from deepchopper_amd import ops

    z = torch.zeros((4, 8))
    for call in (lambda: ops.token_logprobs(z), lambda: ops.gated_scan(z, z, offsets=torch.tensor([0, 4])), lambda: ops.block_norm(z, z)):
        with pytest.raises(ValueError, match="device-resident"):
            call()
