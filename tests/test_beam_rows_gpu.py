"""kd_beam_select over logits whose rows are views into something wider."""
import numpy as np
import pytest

from kandle_b200.core import Tensor
from kandle_b200.model_utils import beam_select
from tests.test_beam_gpu import check

pytestmark = pytest.mark.gpu


def test_one_beam_of_many_is_a_view(backend):
    """[requests, 1, V] out of [requests, beams, V], and one request out of several: the rows are evenly spaced."""
    rng = np.random.default_rng(0)
    all_ = (rng.standard_normal((5, 4, 1000)) * 2.5).astype(np.float32)
    t = Tensor(all_)
    for at in (0, 3):
        check(all_[:, at:at + 1], np.zeros((5, 1), np.float32), 7, beam_select(t.slice([slice(None), slice(at, at + 1), slice(None)]), Tensor(np.zeros((5, 1), np.float32)), 7))
    check(all_[2:3], np.zeros((1, 4), np.float32), 7, beam_select(t.slice([slice(2, 3), slice(None), slice(None)]), Tensor(np.zeros((1, 4), np.float32)), 7))
    check(all_[::2, 1:2], np.zeros((3, 1), np.float32), -1, beam_select(t.slice([slice(None, None, 2), slice(1, 2), slice(None)]), Tensor(np.zeros((3, 1), np.float32)), -1))
