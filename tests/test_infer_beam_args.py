"""Arguments that QatModel.infer_beam refuses before anything runs, on the
host: a model object whose library would fail on any call."""
import numpy as np
import pytest
import torch

from trba_b200.model import Config, QatModel


class _NoCalls:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


def _model(**cfg):
    m = QatModel.__new__(QatModel)
    m.cfg, m.L, m.h = Config(**cfg), _NoCalls(), None
    return m


def test_images_are_checked():
    m = _model(img_w=64, max_len=4)
    good = torch.zeros(2, 3, 32, 64, dtype=torch.int8)
    for exc, word, img in ((TypeError, "int8", good.float()), (TypeError, "int8", good.numpy()), (ValueError, "3 x 32 x 64", good[..., :-2]),
                           (ValueError, "3 x 32 x 64", good[:, :2]), (ValueError, "3 x 32 x 64", good[0]),
                           (ValueError, "3 x 32 x 64", torch.tensor(1, dtype=torch.int8)), (ValueError, "cpu", good)):
        with pytest.raises(exc, match=word):
            m.infer_beam(img, 3)
    for img in (good[..., :-2].numpy(), good[0].numpy(), np.zeros((), np.int8)):
        with pytest.raises(ValueError, match="3 x 32 x 64"):
            m.infer_beam_host(img, 3)
    for beams in (0, 33):
        with pytest.raises(ValueError, match="beams"):
            m.infer_beam(good, beams)
        with pytest.raises(ValueError, match="beams"):
            m.infer_beam_host(good.numpy(), beams)
