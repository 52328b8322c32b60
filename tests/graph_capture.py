"""Capture and replay for tests that need autograd inside the graph.

torch keeps the random state of captured graphs in two tensors of the process;
once a capture under inference mode has created them (other tests do), captures
and replays elsewhere may not write them. So both ends run under inference mode
here, and the captured work outside it.
"""

from __future__ import annotations

import torch


def captured(call):
    """``(graph, call's results)`` after one ordinary call on a side stream."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    grad = torch.is_grad_enabled()
    with torch.inference_mode(), torch.cuda.graph(graph):
        with torch.inference_mode(False), torch.set_grad_enabled(grad):
            held = call()
    return graph, held


def replay(graph):
    with torch.inference_mode():
        graph.replay()
