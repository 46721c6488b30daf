"""CPU tests: arguments of the sequence-layer and scoring operators that deepchopper_amd.ops refuses before it looks at a device."""
import pytest
import torch

from deepchopper_amd import ops

CALLS = {
    "token_logprobs": (lambda a: ops.token_logprobs(a["z"]), ["z"]),
    "gated_scan": (lambda a: ops.gated_scan(a["x"], a["f"], h0=a["h0"]), ["x", "f", "h0"]),
    "block_norm": (lambda a: ops.block_norm(a["y"], a["r"], a["g"], scale=a["s"], post_weight=a["w1"], post_bias=a["b1"], pre_weight=a["w2"], pre_bias=a["b2"]),
                   ["y", "r", "g", "s", "w1", "b1", "w2", "b2"]),
}


@pytest.mark.parametrize("name,leaf", [(n, k) for n, (_, keys) in CALLS.items() for k in keys])
def test_inputs_that_autograd_would_follow_are_refused(name, leaf):
    """Their results would be detached without a word: no gradient would ever reach the leaf."""
    call, keys = CALLS[name]
    a = {k: torch.zeros((2, 3, 4)).requires_grad_(k == leaf) for k in keys}
    with pytest.raises(ValueError, match=f"{name}: an input requires gradients.*{name}_backward"):
        call(a)
    # not where nothing is recorded: these get as far as the device
    with torch.no_grad(), pytest.raises(ValueError, match="device-resident"):
        call(a)
    with torch.inference_mode(), pytest.raises(ValueError, match="device-resident"):
        call(a)
    with pytest.raises(ValueError, match="device-resident"):
        call({k: t.detach() for k, t in a.items()})
