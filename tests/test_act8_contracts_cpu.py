"""What the modules around the 8-bit checkpoints and residual norms decide before any kernel runs, checked without a GPU."""
import pytest
import torch
from torch import nn


@pytest.fixture(scope="module")
def V():
    import vita_amd.nn as v
    return v


class PlainNorm(nn.Module):
    """A layer norm that is no nn.LayerNorm: weight, bias, eps and normalized_shape are all that the kernels ask of one."""

    def __init__(self, dim, eps=1e-5):
        super().__init__()
        self.weight, self.bias, self.eps, self.normalized_shape = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.zeros(dim)), eps, (dim,)


@pytest.mark.parametrize("first,second,bits,want", [
    (nn.LayerNorm, nn.LayerNorm, 16, "_BlockFn"), (PlainNorm, PlainNorm, 16, "_BlockFn"), (PlainNorm, nn.LayerNorm, 16, "_BlockFn"),
    (nn.RMSNorm, nn.LayerNorm, 16, "_BlockActFn"), (nn.LayerNorm, nn.RMSNorm, 16, "_BlockActFn"), (nn.RMSNorm, nn.RMSNorm, 16, "_BlockActFn"),
    (nn.LayerNorm, nn.LayerNorm, 8, "_BlockActFn"), (nn.LayerNorm, nn.RMSNorm, 8, "_BlockActFn")])
def test_both_norms_choose_the_function_of_a_block(V, monkeypatch, first, second, bits, want):
    seen = []
    for name in ("_BlockFn", "_BlockActFn"):
        monkeypatch.setattr(getattr(V, name), "apply", lambda *a, name=name: seen.append(name))
    b = V.Block(16, 2, 4.0, qkv_bias=True, saved_bits=bits)
    b.norm1, b.norm2 = first(16), second(16)
    b.forward_padded(torch.zeros(1, 2, 64))
    assert seen == [want]


@pytest.mark.parametrize("norm,bits,want", [(nn.LayerNorm, 16, "_LayerNormFn"), (PlainNorm, 16, "_LayerNormFn"), (nn.RMSNorm, 16, "_NormActFn"),
                                            (nn.LayerNorm, 8, "_NormActFn"), (PlainNorm, 8, "_NormActFn")])
def test_a_norm_that_ran_before_runs_on_the_same_kernels(V, monkeypatch, norm, bits, want):
    seen = []
    for name in ("_LayerNormFn", "_NormActFn"):
        monkeypatch.setattr(getattr(V, name), "apply", lambda *a, name=name: seen.append(name))
    V.layer_norm_padded(torch.zeros(1, 2, 64), norm(16), bits)
    assert seen == [want]


def test_a_linear_layer_that_keeps_8_bits_refuses_second_derivatives(V):
    """Its backward pass is kernels: with create_graph=True its part would be missing.  Refused before any of them runs."""
    from types import SimpleNamespace
    ctx = SimpleNamespace(bits=8, saved_tensors=(None, None, None), dims=(1, 1, 64, 64, 16, 16), needs_input_grad=(True,) * 6)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="second derivatives"):
        V._LinearFn.backward(ctx, torch.zeros(1, 1, 64))


def test_no_probe_for_a_second_stream_under_capture(V, monkeypatch):
    """The probe waits for an event on the host, which ends a capture; a capture uses one stream anyway.  The next eager forward pass
    probes then, and a stream that was found before is returned under capture too."""
    dev = torch.device("cuda", 0)
    monkeypatch.setattr(V, "_SIDE_STREAMS", {})
    probes, capturing = [], [True]
    monkeypatch.setattr(V, "_concurrent_stream", lambda idx, main: probes.append(idx) or "stream")
    monkeypatch.setattr(torch.cuda, "current_stream", lambda idx=None: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    assert V.ensure_side_stream(dev) is None and probes == [] and V._SIDE_STREAMS == {}
    h = V._Shadows()
    h._build["w"] = (lambda: None, None)
    V.prefetch_shadows(dev)                             # nothing to fork to: the copies are rebuilt where they are used
    assert probes == []
    capturing[0] = False
    assert V.ensure_side_stream(dev) == "stream" and probes == [0]
    capturing[0] = True
    assert V.ensure_side_stream(dev) == "stream" and probes == [0]


@pytest.mark.parametrize("capturing,enabled", [(True, True), (False, False)])
def test_a_failed_backward_pass_does_not_swallow_later_reports(V, monkeypatch, capturing, enabled):
    """An eager Block backward that raised leaves its list of deferred reports behind.  A later one on one stream (as under capture) has no
    join that would hand it on: its accumulated gradients are reported at once."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(V, "_DEFERRED_DONE", [])
    p, seen = nn.Parameter(torch.zeros(1)), []
    monkeypatch.setattr(V, "GRAD_READY", {id(p): seen.append})
    side = V._SideStream(torch.device("cuda", 0), enabled)
    assert not side.on
    side(V.grad_done, p)
    side.join()
    assert len(seen) == 1 and seen[0] is p and V._DEFERRED_DONE is None
