"""AttentionBlock's decays as a part of its state: state dicts, types and devices, without a GPU."""
import copy
import io
import warnings

import pytest
import torch

OWN = [-0.5, -0.001, -3.0, float("-inf")]


def block(**kw):
    import laplacianformer_amd as lf

    return lf.AttentionBlock(32, 4, attention="decay", **kw)


def test_state_dict_carries_the_decays():
    own, other = block(log_decay=OWN), block()
    assert not torch.equal(own._log_decay, other._log_decay)
    buf = io.BytesIO()
    torch.save(torch.nn.Sequential(own).state_dict(), buf)
    buf.seek(0)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        torch.nn.Sequential(other).load_state_dict(torch.load(buf, weights_only=True), strict=True)
    assert torch.equal(other._log_decay, torch.tensor(OWN)) and torch.equal(copy.deepcopy(own)._log_decay, own._log_decay)
    assert "_log_decay" not in dict(own.named_parameters())
    with pytest.raises(RuntimeError, match="size mismatch"):
        import laplacianformer_amd as lf

        lf.AttentionBlock(32, 2, attention="decay").load_state_dict(own.state_dict())


def test_state_dict_without_decays():
    """One saved when they were in none: it loads with a warning, and the block keeps its own."""
    sd = {n: t for n, t in block().state_dict().items() if n != "_log_decay"}
    own = block(log_decay=OWN)
    with pytest.warns(UserWarning, match="_log_decay"):
        own.load_state_dict(sd, strict=True)
    assert torch.equal(own._log_decay, torch.tensor(OWN)) and torch.equal(own.weight, sd["weight"])
    with pytest.raises(RuntimeError, match="Missing key"):
        own.load_state_dict({n: t for n, t in block().state_dict().items() if n != "weight"})


@pytest.mark.parametrize("to", [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                                lambda m: torch.nn.Sequential(m).to("cpu", torch.bfloat16)[0]])
def test_decays_stay_float32(to):
    b = to(block(log_decay=OWN))
    assert b.weight.dtype != torch.float32
    assert b._log_decay.dtype == torch.float32 and torch.equal(b._log_decay, torch.tensor(OWN))
    assert b.to("meta")._log_decay.device.type == "meta"


def test_assigned_state_dict_in_16_bits():
    sd = {n: t.bfloat16() for n, t in block(log_decay=OWN).state_dict().items()}
    b = block()
    b.load_state_dict(sd, assign=True)
    assert b.weight.dtype == torch.bfloat16 and b._log_decay.dtype == torch.float32
    assert torch.equal(b._log_decay, torch.tensor(OWN).bfloat16().float())


def test_other_attentions_have_none():
    import laplacianformer_amd as lf

    for a in ("softmax", "laplacian"):
        b = lf.AttentionBlock(32, 4, attention=a)
        assert not any("log_decay" in n for n in b.state_dict())
        b.half().load_state_dict(lf.AttentionBlock(32, 4, attention=a).state_dict())
