"""Where a module's dropout bits come from: a (seed, offset) pair on its device.

``hc_dropout`` and ``hc_mix_write_norm`` take such a pair as their ``seed``.
A module that drops out holds a ``DropState`` and draws from it:

    with self.bits.drawn(x.device) as seed:
        y = hc_dropout(x, p, seed)

Every draw has its own offset, also when a CUDA graph that holds it is
replayed. A forward that a checkpoint runs again in the backward pass draws what
it drew the first time.
"""

from __future__ import annotations

from collections import OrderedDict
from contextlib import contextmanager

import torch
import torch.distributed as dist
import torch.nn as nn


def _may_run_again() -> bool:
    """Whether a forward that runs now may be one that a backward pass repeats:
    a checkpoint runs it without gradients, or keeps what it saves out of its
    graph by hooks."""
    return not torch.is_grad_enabled() or torch._C._autograd._top_saved_tensors_default_hooks(True) is not None


def _number() -> int:
    return int(torch.randint(1 << 62, (), device="cpu"))


_RANK_STEP = 0x1E3779B97F4A7C15  # odd: no two ranks below 2^62 meet


def _rank() -> int:
    return dist.get_rank() if dist.is_available() and dist.is_initialized() else 0


class DropState(nn.Module):
    """``state``: int64 (seed, offset), seeded from torch's generator and not
    part of the ``state_dict``. Each draw has the state as it is and adds 1 to
    the offset.

    The ranks of a job seed torch alike and drop out different tokens, so with
    ``torch.distributed`` set up before the module is made, each rank's seed is
    its own (rank 0's is the generator's). The state is no buffer:
    DistributedDataParallel would put rank 0's on every rank before each forward.
    It moves with the module, or to where it is first drawn. Ranks that hold the
    same tokens want the same state: set it.

    A checkpoint's second forward runs inside the backward pass, from the same
    state of torch's CPU generator as the first (``preserve_rng_state``, its
    default). So a first forward that may be repeated takes a number from that
    generator and files its own (seed, offset) under it; inside a backward pass
    the number that comes again finds them, and the state stays as it is. What
    is not found is refused with an error, since other bits than the loss's
    would give gradients of something else: a checkpoint with
    ``preserve_rng_state=False``, one whose first forward lies more than
    ``KEPT`` draws of this module back, or two forwards that began from one
    state of the generator and were both yet to be repeated. The number is
    taken only where a repetition is possible, so that a plain step leaves the
    generator alone."""

    KEPT = 256

    def __init__(self, seeded: bool = True):
        super().__init__()
        seed = torch.randint(1 << 62, (1,)) if seeded else torch.zeros(1, dtype=torch.int64)
        if seed.is_meta:  # a module without memory yet
            seed = torch.randint(1 << 62, (1,), device="cpu")
        if seeded and _rank() > 0:
            seed = (seed + _rank() * _RANK_STEP % (1 << 62)) % (1 << 62)  # the sum stays below 2^63
        self.state = torch.cat([seed, torch.zeros_like(seed)])
        self._filed = OrderedDict()  # number -> [(seed, offset), drawn again, two of them]

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self._move(fn(self.state).device)
        return self

    def _move(self, device: torch.device) -> None:
        if device.type != "meta":
            with torch.inference_mode(False):  # which makes tensors that no later step could move on
                self.state = self.state.to(device)

    def __getstate__(self):  # of a copy: its own draws
        return {**self.__dict__, "_filed": OrderedDict()}

    def _file(self, drawn: torch.Tensor) -> None:
        number = _number()
        before = self._filed.pop(number, None)
        self._filed[number] = [drawn, False, before is not None and (before[2] or not before[1])]
        while len(self._filed) > self.KEPT:
            self._filed.popitem(last=False)

    def _find(self) -> torch.Tensor:
        entry = self._filed.get(_number())
        if entry is None:
            raise RuntimeError(
                "dropout inside a backward pass whose first forward is not known: a recomputed forward has to begin from the "
                "random state of the first one (torch.utils.checkpoint with preserve_rng_state=True, its default)")
        if entry[2]:
            raise RuntimeError(
                "dropout inside a backward pass with two first forwards that began from the same random state: give each its "
                "own (do not reset torch's generator between them)")
        entry[1] = True
        return entry[0]

    @contextmanager
    def drawn(self, device: torch.device):
        """The (seed, offset) of one forward, on `device`."""
        self._move(device)
        if torch._C._current_graph_task_id() != -1:  # a backward pass is running on this thread
            yield self._find()
        elif _may_run_again():
            drawn = self.state.clone()
            self._file(drawn)
            yield drawn
            self.state[1].add_(1)
        else:
            yield self.state
            self.state[1].add_(1)
