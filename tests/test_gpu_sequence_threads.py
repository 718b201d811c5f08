"""GPU tests of the sequence operators where calls meet: threads, each operator in every way of
launching, counted so that a call that fails in its thread fails the test; workspaces that are
certainly used; many streams of one frame."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import sequence_cases as cases
from fast_gpu_asr_b200 import (gated_linear_recurrence, gated_linear_recurrence_backward,
                               group_norm_activation, group_norm_activation_backward,
                               normalization, recurrence)
from oracle import sequence_oracle as oracle

pytestmark = pytest.mark.gpu

CALLS = 20


def norm_call(n, t, c, groups, dtype, seed):
    x, w, b, dout = (cases.to_cuda(v, dtype) for v in cases.norm_inputs(n, t, c, dtype, seed))
    lens = torch.from_numpy(cases.mixed_lengths(n, t, seed)).cuda()

    def call():
        out, mean, rstd = group_norm_activation(x, lens, w, b, groups, return_statistics=True)
        return (out, mean, rstd, *group_norm_activation_backward(dout, x, lens, w, b, mean, rstd))

    return call


def recurrence_call(n, t, c, dtype, seed):
    x, gate, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, dtype, seed)
    x, gate, dout = (cases.to_cuda(v, dtype) for v in (x, gate, dout))
    initial, dfinal = (cases.to_cuda(v, "float32") for v in (initial, dfinal))
    lens = torch.from_numpy(cases.mixed_lengths(n, t, seed)).cuda()

    def call():
        got = gated_linear_recurrence(x, gate, lens, initial, return_states=True)
        return (*got, *gated_linear_recurrence_backward(dout, x, gate, lens, got[2], dfinal))

    return call


@pytest.mark.parametrize("kinds", ["norm", "recurrence", "both"])
def test_calls_from_threads(kinds):
    """Two threads a problem, each on a stream of its own. Among the norms are clusters, streams
    and rows that start anywhere; among the recurrences walks that several blocks divide."""
    calls = []
    if kinds in ("norm", "both"):
        calls += [norm_call(3, 900, 64, 1, "float16", 0), norm_call(4, 100, 96, 12, "bfloat16", 1),
                  norm_call(1, 12000, 40, 1, "float32", 2), norm_call(3, 200, 129, 3, "float16", 3)]
    if kinds in ("recurrence", "both"):
        calls += [recurrence_call(1, 5000, 64, "float16", 4),
                  recurrence_call(3, 700, 65, "bfloat16", 5),
                  recurrence_call(2, 3000, 40, "float32", 6),
                  recurrence_call(40, 60, 128, "float16", 7)]
    problems = [(call, call()) for call in calls]
    torch.cuda.synchronize()
    done, wrong = [], []

    def work(call, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(CALLS):
                    got = call()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want)):
                        raise AssertionError("other bits than the first call's")
                    done.append(1)
        except BaseException as e:  # noqa: BLE001 - a thread's own exception would go unseen
            wrong.append(e)

    threads = [threading.Thread(target=work, args=p) for p in problems for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong, wrong
    assert len(done) == CALLS * len(threads)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_a_workspace_that_is_used(dtype):
    """Streams and divided walks: their query is above zero, and nothing past it is written."""
    norm = [cases.to_cuda(v, dtype) for v in cases.norm_inputs(1, 12000, 40, dtype, 6)]
    lens = torch.tensor([11987], dtype=torch.int32, device="cuda")
    x, w, b, dout = norm
    rec = cases.recurrence_inputs(1, 5000, 64, dtype, 6)
    rx, gate, rdout = (cases.to_cuda(v, dtype) for v in rec[:3])
    rlens = torch.tensor([4990], dtype=torch.int32, device="cuda")
    _, mean, rstd = group_norm_activation(x, lens, w, b, 1, return_statistics=True)
    _, _, states = gated_linear_recurrence(rx, gate, rlens, return_states=True)
    for size, call in (
            (normalization.group_norm_activation_workspace_size(x, lens, w, b, 1),
             lambda **k: (group_norm_activation(x, lens, w, b, 1, **k),)),
            (normalization.group_norm_activation_backward_workspace_size(x, lens, w, b, 1),
             lambda **k: group_norm_activation_backward(dout, x, lens, w, b, mean, rstd, **k)),
            (recurrence.gated_linear_recurrence_workspace_size(rx, rlens),
             lambda **k: gated_linear_recurrence(rx, gate, rlens, **k)),
            (recurrence.gated_linear_recurrence_backward_workspace_size(rx, rlens),
             lambda **k: gated_linear_recurrence_backward(rdout, rx, gate, rlens, states, **k))):
        assert size > 0
        room = torch.full((size + 256,), 171, dtype=torch.uint8, device="cuda")
        want, got = call(), call(workspace=room[:size])
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        assert torch.all(room[size:] == 171) and not torch.all(room[:size] == 171)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_many_streams_of_one_frame(dtype):
    """Steps of 1024 streams of aligned rows, their state updated in place, in a graph and not."""
    n, t, c = 1024, 3, 512
    x, gate, _, initial, _ = cases.recurrence_inputs(n, t, c, dtype, 19)
    gx, gg = cases.to_cuda(x, dtype), cases.to_cuda(gate, dtype)
    lengths = np.ones(n, np.int32)
    lengths[::7] = 0  # streams that have no frame in this step
    lens = torch.from_numpy(lengths).cuda()
    state, in_graph = (cases.to_cuda(initial, "float32") for _ in range(2))
    step_x, step_g = gx[:, :1].contiguous(), gg[:, :1].contiguous()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured, _ = gated_linear_recurrence(step_x, step_g, lens, in_graph, final_state=in_graph)
    in_graph.copy_(cases.to_cuda(initial, "float32"))
    expected = oracle.gated_linear_recurrence(x, gate, lengths * t, initial)
    bounds = cases.recurrence_bounds(x, gate, lengths * t, initial, expected, dtype)
    for i in range(t):
        step_x.copy_(gx[:, i:i + 1])
        step_g.copy_(gg[:, i:i + 1])
        g.replay()
        out, final = gated_linear_recurrence(step_x, step_g, lens, state, final_state=state)
        assert final is state and torch.equal(out, captured) and torch.equal(state, in_graph)
        cases.assert_within(cases.host(out)[:, 0], expected[0][:, i], bounds[0][:, i], i)
    cases.assert_within(cases.host(state), expected[1], bounds[1])
    assert torch.equal(state[::7], cases.to_cuda(initial, "float32")[::7])
