"""Calls that the sequence operators refuse before anything is launched, without a device: torch's
view of the current device and stream is replaced."""

from __future__ import annotations

import types

import pytest
import torch
from torch.autograd import forward_ad

from fast_gpu_asr_b200 import (_call, _lib, gated_linear_recurrence, gated_linear_recurrence_backward,
                               group_norm_activation, group_norm_activation_backward,
                               normalization, recurrence)


def calls(x, **options):
    """Each operator on tensors shaped after ``x`` [N, T, C]."""
    n, t, c = x.shape
    lens, w = torch.zeros(n, dtype=torch.int32), x.new_ones(c)
    stats, states = torch.zeros(n, 1), torch.zeros(n, -(-t // 64), c)
    return (lambda: group_norm_activation(x, lens, w, w, 1, **options),
            lambda: group_norm_activation_backward(x, x, lens, w, w, stats, stats, **options),
            lambda: gated_linear_recurrence(x, x, lens, **options),
            lambda: gated_linear_recurrence_backward(x, x, x, lens, states, **options))


def test_a_stream_of_another_device(monkeypatch):
    """It would make its device the current one, and the kernels read the tensors from there."""
    def entered(stream):
        raise AssertionError("the stream's device was made the current one")

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "stream", entered)
    monkeypatch.setattr(_call, "_torch_stream", lambda s: s)
    stream = types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=0)
    for call in calls(torch.zeros(2, 3, 4), stream=stream):
        with pytest.raises(ValueError, match="stream is on cuda:1, the current device is cuda:0"):
            call()


def test_forward_mode_tangents(monkeypatch):
    """They would be lost. (A tensor on the CPU is on device -1, which stands for the current one
    here; nothing is launched.)"""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(_call, "_current_stream", lambda device: 0)

    def launched(self, *args):
        raise AssertionError("the call went on to its launch")

    monkeypatch.setattr(_call.Operator, "_plan", launched)
    x = torch.zeros(2, 3, 4)
    with forward_ad.dual_level():
        for call in calls(forward_ad.make_dual(x, torch.ones_like(x))):
            with pytest.raises(ValueError, match="carries a forward-mode tangent"):
                call()
        with torch.no_grad():
            for call in calls(forward_ad.make_dual(x, torch.ones_like(x))):
                with pytest.raises(ValueError, match="carries a forward-mode tangent"):
                    call()
        for call in calls(x):
            with pytest.raises(AssertionError, match="went on"):
                call()


@pytest.mark.parametrize("n,t", [(2 ** 31 - 1, 1), (2, 2 ** 30 - 1), (1, 2 ** 30)])
def test_the_most_frames_of_a_batch(library, n, t):
    """The kernels' loops over frames, utterances and blocks take what the checks let through: all
    their counts are below 2^31 and a step past the last one below 2^32."""
    d, F32 = _lib.TensorDesc.make, _lib.FGA_FLOAT
    w = d(F32, (1,))
    for n, status in ((n, 0), (2 ** 31 // t + 1, 4)):
        a, lens, stats = d(F32, (n, t, 1)), d(_lib.FGA_INT32, (n,)), d(F32, (n, 1))
        states = d(F32, (n, -(-t // 64), 1))
        assert normalization.group_norm_activation_check(
            [a, lens, w, w], [a, stats, stats], 1, 1e-5, "silu") == status
        assert normalization.group_norm_activation_backward_check(
            [a, a, lens, w, w, stats, stats], [a, w, w], "silu") == status
        assert recurrence.gated_linear_recurrence_check(
            [a, a, lens, stats], [a, stats, states]) == status
        assert recurrence.gated_linear_recurrence_backward_check(
            [a, a, a, lens, states, stats], [a, a, stats]) == status
