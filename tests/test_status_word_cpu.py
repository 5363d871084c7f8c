"""No-GPU check: a status mirror made in inference mode serves calls outside of it."""
import torch

from paraattention_b200._status import StatusMirror


def test_a_mirror_made_in_inference_mode_can_be_written_later():
    word = torch.zeros(1, dtype=torch.int32)
    with torch.inference_mode():
        m = StatusMirror(word)
    m.refresh()
    m.check_now()
    m.reset()
