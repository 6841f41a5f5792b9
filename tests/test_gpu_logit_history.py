"""A history without a pitch is refused: with a pitch of nothing it would count for nothing."""

import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu


def test_a_history_has_a_pitch(ctx):
    dev = lambda values, dtype: torch.tensor(values, dtype=dtype, device="cuda")
    logits, out = torch.ones(1, 8, device="cuda"), torch.full((1, 8), 9.0, device="cuda")
    starts, lengths, history = dev([0, 1], torch.int32), dev([2], torch.int32), dev([[3, 5]], torch.int64)
    penalties = dev([[2.0, 0.0, 0.0]], torch.float32)
    torch.cuda.synchronize()
    call = lambda **kw: ctx.adjust_logits(logits.data_ptr(), 8, out.data_ptr(), starts.data_ptr(), 1, 1, penalties=penalties.data_ptr(),
                                          history=history.data_ptr(), history_lengths=lengths.data_ptr(), **kw)
    with pytest.raises(B.BackendError) as e:
        call()
    assert e.value.code == B.INVALID
    ctx.synchronize()
    assert (out == 9.0).all()
    call(history_pitch=2)
    ctx.synchronize()
    assert out.tolist() == [[1.0, 1.0, 1.0, 0.5, 1.0, 0.5, 1.0, 1.0]]
    # longer than its pitch: the pitch's
    lengths.fill_(7)
    torch.cuda.synchronize()
    call(history_pitch=1)
    ctx.synchronize()
    assert out.tolist() == [[1.0, 1.0, 1.0, 0.5, 1.0, 1.0, 1.0, 1.0]]
