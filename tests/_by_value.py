"""A process queue that carries tensors by value.

``torch.multiprocessing`` hands over file descriptors that the receiver fetches from the sender, which must still run then: a worker
that puts its results and ends may be gone (ConnectionResetError)."""
from __future__ import annotations

import io
import multiprocessing.queues

import torch


class Queue(multiprocessing.queues.Queue):
    def put(self, obj, *args, **kw):
        data = io.BytesIO()
        torch.save(obj, data)
        super().put(data.getvalue(), *args, **kw)

    def get(self, *args, **kw):
        return torch.load(io.BytesIO(super().get(*args, **kw)), weights_only=False)


def context_with(ctx):
    """``ctx`` with its queues replaced."""
    ctx.Queue = lambda maxsize=0: Queue(maxsize, ctx=ctx)
    return ctx
