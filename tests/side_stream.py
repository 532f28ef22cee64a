"""A stream beside the current one for the training operators' tests: the one that torch captures graphs on.

HIP maps the streams of a process onto a few hardware queues (4 by default), and streams that share one run in the order of their
work. Tests of overlap, as of save-backs under compute, depend on how many streams there are; these tests add none to the
one that every capture without a stream of its own uses."""
from __future__ import annotations

import torch


def side_stream() -> torch.cuda.Stream:
    if torch.cuda.graph.default_capture_stream is None:
        torch.cuda.graph.default_capture_stream = torch.cuda.Stream()
    return torch.cuda.graph.default_capture_stream
