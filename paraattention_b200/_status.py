"""Device status words and their host mirrors.

Every bounded wait in the kernels reports a timeout by writing a ``pa_device_status`` code into a
device word and makes every later launch that is given the same word return at its entry, so a
stuck exchange can never hang a GPU - but it also means that from then on results are garbage
until somebody looks at the word. ``StatusMirror`` makes the host look without adding a device
synchronisation to the call path: after each launch the word is copied (asynchronously, 4 bytes)
into pinned host memory, and before each launch the host copy - which by then holds the state
after some earlier launch - is read. A timeout therefore surfaces as a ``PaError(PA_ETIMEDOUT)``
on one of the next calls (at the latest after the next synchronisation), where the reference's
NCCL path would raise or abort on a stuck collective. ``reset()`` clears both words.
"""
from __future__ import annotations

from typing import Dict, List

import torch

from . import _lib as L


class StatusMirror:
    def __init__(self, word: torch.Tensor):
        assert word.dtype == torch.int32 and word.numel() == 1
        self.word = word
        # (an ordinary tensor, also if the first call is made in inference mode: later ones write to it)
        with torch.inference_mode(False):
            host = torch.zeros(1, dtype=torch.int32)
            # (pinning needs a CUDA runtime; a CPU word - the unit tests - gets a plain host copy)
            self.host = host.pin_memory() if word.device.type == "cuda" else host

    def check(self) -> None:
        """Raise if an earlier launch reported a timed-out wait. Reads host memory only."""
        code = int(self.host[0])
        if code != 0:
            raise L.PaError(L.PA_ETIMEDOUT,
                            L.DEV_STATUS_NAMES.get(code, f"device status {code}") +
                            " (the status word is sticky: call reset() once the cause is dealt with)")

    def refresh(self) -> None:
        """Queue a copy of the device word to the host mirror on the current stream."""
        self.host.copy_(self.word, non_blocking=True)

    def check_now(self) -> None:
        """Synchronising form: read the device word itself."""
        self.host.copy_(self.word)
        self.check()

    def reset(self) -> None:
        """Clear both words. Waits for the device: launches in flight that found the old code report it first."""
        self.word.zero_()
        if self.word.device.type == "cuda":
            torch.cuda.synchronize(self.word.device)
        self.host.zero_()


_single: Dict[int, StatusMirror] = {}
_in_graphs: List[StatusMirror] = []  # made by first calls inside a capture; graphs hold their addresses


def single_gpu_status(device: torch.device) -> StatusMirror:
    """The status word the single-GPU attention ops of this process share on ``device``."""
    m = _single.get(device.index)
    if m is not None:
        return m
    with torch.cuda.device(device), torch.inference_mode(False):
        if torch.cuda.is_current_stream_capturing():
            # This word is filled by the graph, in front of the launches that read it: it is the graph's alone.
            m = StatusMirror(torch.zeros(1, dtype=torch.int32, device=device))
            _in_graphs.append(m)
            return m
    # Launches on any stream read the word without waiting for this one, so it is filled before its address is
    # known: on a stream of its own, which may be waited for while this one is busy.
    stream = torch.cuda.Stream(device)
    with torch.cuda.stream(stream), torch.inference_mode(False):
        word = torch.zeros(1, dtype=torch.int32, device=device)
    stream.synchronize()
    m = _single[device.index] = StatusMirror(word)
    return m


def all_mirrors():
    return [*_single.values(), *_in_graphs]
