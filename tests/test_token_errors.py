"""What the status word's codes raise. No GPU: the word lies on the host."""
import pytest
import torch

from ccfuser_b200 import MoECommError, TokenIndexError
from ccfuser_b200.ops.gemm import Workspace


def _raised(word):
    ws = Workspace(torch.device("cpu"))
    ws.status[0] = word
    with pytest.raises(Exception) as e:
        ws.check("test")
    assert ws.status.tolist() == [0, 0]
    return e.value


def test_a_bad_id_is_no_lost_peer():
    e = _raised(7 << 8 | 5)
    assert isinstance(e, TokenIndexError) and isinstance(e, IndexError) and isinstance(e, RuntimeError)
    assert not isinstance(e, MoECommError) and "token 7 " in str(e)
    assert isinstance(_raised(2), MoECommError)


def test_the_number_of_a_late_token():
    assert "token 8388606 lies" in str(_raised(8388606 << 8 | 5))
    assert "token 8388607 or a later one" in str(_raised(8388607 << 8 | 5))
