"""Launches of the library's entries, and their index errors through pinned host memory.

The host's share counts where a call's kernels take ten microseconds: one function makes the call on
the device's current stream, with the device made current and the region timed only where that is
asked for.

A kernel that meets an index it cannot compute with writes NaN and sets a word here: a plain store,
which only a bad index ever makes, so a launch needs no device flag to be cleared before it and
copied after it, just an event behind it. The words go back to a pool when their owner is dropped, and
are handed out again once their event has passed: a launch whose owner is gone may still write.
"""

from __future__ import annotations

import contextlib
from collections import defaultdict, deque

import torch

from aspec_amd import _lib, _timing

# the words, in the order of include/aspec_amd.h
_MESSAGES = (
    "teacher index out of range: every target index must address a row of the teacher table",
    "cross-entropy target out of range: targets must lie in [0, vocab) or equal ignore_index",
    "token id out of range: token ids must lie in [0, vocab) or equal ignore_index",
    "teacher token out of range: a teacher row's tokens must lie in [0, vocab), or be -1 for an unused slot",
    "teacher token repeated: a teacher row's tokens must be distinct",
)
_pool = defaultdict(deque)


class IndexFlags:
    """The words of one launch on `device`: `ptr` goes to the kernel, `record` follows the launch on its
    stream, `raise_if_bad` waits for it and raises ValueError where an index was bad."""

    def __init__(self, device: torch.device):
        self.device, self._home = device, _pool[device.index]
        self._slot = None
        for _ in range(min(2, len(self._home))):  # the oldest first; one still pending goes to the end
            with contextlib.suppress(IndexError):
                slot = self._home.popleft()
                if slot[2].query():
                    self._slot = slot
                    break
                self._home.append(slot)
        if self._slot is None:
            words = torch.zeros(len(_MESSAGES), dtype=torch.int32, pin_memory=True)
            self._slot = (words, words.numpy(), torch.cuda.Event(), words.data_ptr())
        self._slot[1].fill(0)
        self.ptr = self._slot[3]

    def record(self, stream: torch.cuda.Stream) -> None:
        self._slot[2].record(stream)

    def raise_if_bad(self) -> None:
        self._slot[2].synchronize()
        if self._slot[1].any():
            raise ValueError(_MESSAGES[int(self._slot[1].argmax())])

    def __del__(self):
        if self._slot is not None:
            self._home.append(self._slot)


def _capturing(device: torch.device) -> bool:
    """Whether the device's current stream is being captured into a graph."""
    if torch.cuda.current_device() == device.index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def index_flags(wanted: bool, device: torch.device) -> IndexFlags | None:
    """The flags of a launch whose indices are to be checked. None where nothing can read them: the
    caller wants no check, or the launch is captured into a graph, whose replays no host follows."""
    if not wanted or _capturing(device):
        return None
    return IndexFlags(device)


# From this many bytes of logits a call that has to read its check before it returns has its indices
# checked by a kernel of their own, ahead of the logits' pass, and waits for that one: the pass then runs
# on while the host prepares the next call. bf16 rows of 32000, us a call (a call that the GPU is waited
# for behind): 2048 of them, losses and gradient, 64 (100) so and 92 (96) with the check in the pass;
# 256 of them 46 (63) and 53 (59).
CHECK_FIRST_BYTES = 1 << 25


def check_first(flags: IndexFlags | None, logits: torch.Tensor) -> bool:
    return flags is not None and logits.numel() * logits.element_size() >= CHECK_FIRST_BYTES


def settle(flags: IndexFlags | None) -> None:
    """Reads a deferred check behind the launches that it was deferred for."""
    if flags is not None and not _capturing(flags.device):
        flags.raise_if_bad()


def launch(region: str, device: torch.device, flags: IndexFlags | None, entry: str, *args) -> None:
    """`entry(*args, stream)` on the device's current stream; `flags` are recorded behind it."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return launch(region, device, flags, entry, *args)
    stream = torch.cuda.current_stream(device)
    if _timing._enabled:
        with _timing.region(region):
            _lib.call(entry, *args, stream.cuda_stream)
    else:
        _lib.call(entry, *args, stream.cuda_stream)
    if flags is not None:
        flags.record(stream)
