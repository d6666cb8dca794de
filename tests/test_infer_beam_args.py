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
    m.cfg, m.L, m.h, m.device = Config(**cfg), _NoCalls(), None, 0
    return m


def test_images_are_checked():
    m = _model(img_w=64, max_len=4)
    good = torch.zeros(2, 3, 32, 64, dtype=torch.int8)
    for exc, word, img in ((TypeError, "int8", good.float()), (TypeError, "int8", good.numpy()), (ValueError, "3 x 32 x 64", good[..., :-2]),
                           (ValueError, "3 x 32 x 64", good[:, :2]), (ValueError, "3 x 32 x 64", good[0]),
                           (ValueError, "3 x 32 x 64", torch.tensor(1, dtype=torch.int8)), (ValueError, "the model is on cuda:0", good)):
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


def test_calls_go_to_the_models_device(monkeypatch):
    """A model made on one device runs there whatever device is current."""
    m = _model(img_w=64, max_len=4)
    m.device, now, used = 1, [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            now.append(self.index)

        def __exit__(self, *exc):
            now.pop()

    class Lib:
        def trba_model_infer_beam_host(self, h, img, b, beams, seq, lens, scores, stream):
            used.append(now[-1])
            return 0

    m.L = Lib()
    monkeypatch.setattr(torch.cuda, "device", Device)
    m.infer_beam_host(np.zeros((2, 3, 32, 64), np.int8), 3)
    assert used == [1] and now == [0]
    from torch._subclasses.fake_tensor import FakeTensorMode
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[-1])
    with FakeTensorMode():
        there, here = (torch.zeros(2, 3, 32, 64, dtype=torch.int8, device=f"cuda:{i}") for i in (1, 0))
    with pytest.raises(ValueError, match="images are on cuda:0, the model is on cuda:1"):
        m.infer_beam(here, 3)
    monkeypatch.setattr(QatModel, "infer_beam", _spied(QatModel.infer_beam, now, used))
    with pytest.raises(_Stop):
        m.infer_beam(there, 3)
    assert used == [1, 0, 1] and now == [0]


class _Stop(Exception):
    pass


def _spied(call, now, used):
    def spy(self, *args):
        used.append(now[-1])
        if now[-1] == self.device:
            raise _Stop
        return call(self, *args)
    return spy
