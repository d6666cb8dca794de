"""Beam search over the recogniser's own decoder (trba_model_infer_beam):
against a search by the oracle that carries every beam's token list along and
recomputes its logits from the start at every step; and, with one beam, against
greedy decoding."""
import sys

import numpy as np
import pytest

from conftest import REPO
from test_infer_gpu import _pair

sys.path.insert(0, str(REPO / "oracle"))
import decode_oracle as do  # noqa: E402
import step_oracle as so  # noqa: E402

pytestmark = pytest.mark.gpu


def search(orc, cfg, img, K):
    """[line][beam] = (tokens before eos, f64 score), best first."""
    b = img.shape[0]
    enc, t = orc.encode(img)
    paths = [[[] for _ in range(K)] for _ in range(b)]
    scores = np.full((b, K), -np.inf)
    scores[:, 0] = 0
    fin = np.zeros((b, K), bool)
    for _ in range(cfg.steps):
        logits = orc.decode_logits(enc, b, t, [(i, p) for i in range(b) for p in paths[i]])
        # the device rounds the running score to f32 at every step
        s, tok, par, fin = do.beam_select(logits, scores.astype(np.float32), fin, cfg.eos)
        scores = s.astype(np.float32).astype(np.float64)
        paths = [[paths[i][par[i, k]] + [int(tok[i, k])] for k in range(K)] for i in range(b)]
    cut = [[p[:p.index(cfg.eos)] if cfg.eos in p else p for p in line] for line in paths]
    return cut, scores


@pytest.mark.parametrize("K", [1, 3, 8])
@pytest.mark.parametrize("geom,B,steps", [(dict(img_w=64, max_len=4), 8, 3), (dict(img_w=96, max_len=9), 3, 2)],
                         ids=["32x64_b8", "32x96_b3"])
def test_beam_search_matches_oracle(geom, B, steps, K, lib, cuda):
    import torch
    ocfg, orc, gm = _pair(geom, B, seed=78, train_steps=steps)
    img, *_ = so.make_batch(ocfg, B, seed=1235)
    want, want_s = search(orc, ocfg, img, K)
    dev = torch.from_numpy(np.ascontiguousarray(img)).cuda()
    seq, lengths, scores = (x.cpu().numpy() for x in gm.infer_beam(dev, K))
    # a step's score is off by at most 2^-19 and half an f32 step (see the
    # selection's tests), so a path's by that times its steps; a beam whose
    # oracle score is nearer than that to another's may change places with it
    tol = ocfg.steps * (2.0 ** -19 + 2.0 ** -24 * np.abs(want_s).max())
    assert np.abs(scores - want_s).max() <= tol
    for i in range(B):
        apart = np.diff(want_s[i]) < -2 * tol
        clear = np.concatenate([[True], apart]) & np.concatenate([apart, [False]])
        for k in range(K):
            n = lengths[i, k]
            assert (seq[i, k, n:] == ocfg.pad).all()
            got = seq[i, k, :n].tolist()
            if clear[k]:
                assert got == want[i][k]
            elif k + 1 < K:
                assert got in want[i]
    host = gm.infer_beam_host(img, K)
    assert [[t for t, _ in line] for line in host] == [[seq[i, k, :lengths[i, k]].tolist() for k in range(K)] for i in range(B)]
    assert np.array_equal(np.array([[s for _, s in line] for line in host], np.float32), scores)
    other, *_ = so.make_batch(ocfg, B, seed=4)
    gm.infer_beam_host(other[:2], K + 1)  # an unrelated call in between, smaller and larger, leaves no trace
    again = gm.infer_beam(dev, K)
    assert np.array_equal(again[0].cpu().numpy(), seq) and np.array_equal(again[2].cpu().numpy(), scores)
    assert lib.trba_last_error() == 0, lib.trba_last_error_string()


def test_one_beam_is_greedy_until_eos(lib, cuda):
    import torch
    ocfg, _, gm = _pair(dict(img_w=160, max_len=20), 4, seed=77, train_steps=2)
    img, *_ = so.make_batch(ocfg, 4, seed=1234)
    dev = torch.from_numpy(np.ascontiguousarray(img)).cuda()
    greedy = gm.infer(dev)
    seq, lengths, _ = (x.cpu().numpy() for x in gm.infer_beam(dev, 1))
    for i in range(4):
        g = greedy[:, i].tolist()
        g = g[:g.index(ocfg.eos)] if ocfg.eos in g else g
        assert seq[i, 0, :lengths[i, 0]].tolist() == g
    assert np.array_equal(gm.infer(dev), greedy)  # the greedy path is as it was


def test_expert_runner_decodes_with_beams(lib, cuda):
    """Serving: the best beam of every line, whatever the decoding batch."""
    import torch
    import trba_b200.mope as mp
    run = mp.ExpertRunner(mp.default_experts()[1], batch=5, seed=11)
    ocfg = so.Config(img_w=96, max_len=5)
    img, *_ = so.make_batch(ocfg, 12, seed=31)
    dev = torch.from_numpy(np.ascontiguousarray(img)).cuda()
    lists = run.decode_beam(dev, 4)
    assert len(lists) == 12
    whole = [run.model.infer_beam(dev[s:s + 5], 4) for s in range(0, 12, 5)]
    for s, (seq, lengths, scores) in zip(range(0, 12, 5), whole):
        assert (scores[:, :-1] >= scores[:, 1:]).all()
        for i in range(seq.shape[0]):
            assert lists[s + i] == seq[i, 0, :lengths[i, 0]].tolist()
    with pytest.raises(ValueError, match="beams"):
        run.model.infer_beam(dev[:1], 33)
    with pytest.raises(RuntimeError, match="infer_beam"):
        run.model.infer_beam(dev, 2)  # more lines than the model was made for
    run.close()


def test_captured_search_outlives_growth(lib, cuda):
    """A search captured into a graph replays on buffers of its own size after
    calls that needed more; the first call of a size is refused in a capture."""
    import torch
    ocfg, _, gm = _pair(dict(img_w=64, max_len=4), 8, seed=78, train_steps=1)
    imgs = [torch.from_numpy(np.ascontiguousarray(so.make_batch(ocfg, 8, seed=s)[0])).cuda() for s in (5, 6)]
    held = lambda: int(lib.trba_model_device_bytes(gm.h))  # noqa: E731
    none = held()
    want = [gm.infer_beam(x[:4], 3) for x in imgs]
    small = held()
    torch.cuda.synchronize()
    buf = imgs[0][:4].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gm.infer_beam(buf, 3)
    assert held() == small
    wide = gm.infer_beam(imgs[1], 8)
    # the small call's block is still there, beside one for (8 x 8) / (4 x 3) as many beams
    assert small > none and held() - small >= 5 * (small - none)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        kept = buf + 0
        with pytest.raises(RuntimeError, match="before its capture"):
            gm.infer_beam(imgs[0], 32)
    for x, w in zip(imgs, want):
        buf.copy_(x[:4])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, w))
    other.replay()
    assert torch.equal(kept, buf)
    assert all(torch.equal(a, b) for a, b in zip(gm.infer_beam(imgs[1], 8), wide))
    assert lib.trba_last_error() == 0, lib.trba_last_error_string()


def test_search_keeps_no_more_than_it_uses(lib, cuda):
    """Device memory of a first search: two sets of h and c, logits, scores,
    the history's tokens and parents, finished (parts of 256 bytes; 130 classes
    need no workspace)."""
    import torch
    ocfg, _, gm = _pair(dict(img_w=64, max_len=4), 8, seed=78, train_steps=0)
    before = int(lib.trba_model_device_bytes(gm.h))
    img = torch.from_numpy(np.ascontiguousarray(so.make_batch(ocfg, 8, seed=5)[0])).cuda()
    gm.infer_beam(img[:4], 3)
    rows = 4 * 3
    parts = [rows * ocfg.hidden * 4] * 4 + [rows * ocfg.classes * 4, rows * 4] + [rows * ocfg.steps * 4] * 2 + [rows]
    assert int(lib.trba_model_device_bytes(gm.h)) - before == sum(-(-p // 256) * 256 for p in parts)


def test_search_on_another_stream(lib, cuda):
    """Results belong to the stream that writes them: their memory, once
    dropped, is not handed to the current one."""
    import ctypes as C
    import torch
    ocfg, _, gm = _pair(dict(img_w=64, max_len=4), 8, seed=78, train_steps=1)
    img = torch.from_numpy(np.ascontiguousarray(so.make_batch(ocfg, 8, seed=5)[0])).cuda()
    want = gm.infer_beam(img, 3)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    for handle in (st.cuda_stream, C.c_void_p(st.cuda_stream)):
        got = gm.infer_beam(img, 3, stream=handle)
        st.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.synchronize()
        like, ptrs = [(t.shape, t.dtype) for t in got], {t.data_ptr() for t in got}
        del got
        kept = [torch.empty(s, dtype=d, device="cuda") for _ in range(40) for s, d in like]
        assert not ptrs & {t.data_ptr() for t in kept}
        with torch.cuda.stream(st):
            assert ptrs & {torch.empty(s, dtype=d, device="cuda").data_ptr() for s, d in like}
    got = gm.infer_beam(img, 3, stream=0)  # the default stream's handle
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert lib.trba_last_error() == 0


def test_expert_runner_on_another_stream(lib, cuda):
    """The stream waits for images that the current one is still to write."""
    import torch
    import trba_b200.mope as mp
    run = mp.ExpertRunner(mp.default_experts()[1], batch=5, seed=11)
    ocfg = so.Config(img_w=96, max_len=5)
    img = torch.from_numpy(np.ascontiguousarray(so.make_batch(ocfg, 12, seed=31)[0])).cuda()
    search, seen = run.model.infer_beam, []

    def scores(imgs, stream=None):  # (an untrained model's tokens hardly depend on the images; its scores do)
        seen.clear()
        lists = run.decode_beam(imgs, 4, stream=stream)
        return lists, torch.cat([r[2] for r in seen]).cpu().numpy()

    run.model.infer_beam = lambda *a, **k: seen.append(search(*a, **k)) or seen[-1]
    want, want_s = scores(img)
    _, zero_s = scores(torch.zeros_like(img))
    assert (zero_s != want_s).all()  # what it would read otherwise
    st = torch.cuda.Stream()
    late, busy = torch.zeros_like(img), torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):  # several ms of work ahead of the images
        busy = torch.tanh(busy @ busy)
    late.copy_(img)
    got, got_s = scores(late, st.cuda_stream)
    assert got == want and np.array_equal(got_s, want_s)
    run.close()


def test_images_that_are_views(lib, cuda):
    """Every other image of a batch, images with a gap between rows, and the
    lines as plain rows of bytes."""
    import torch
    ocfg, _, gm = _pair(dict(img_w=64, max_len=4), 8, seed=78, train_steps=1)
    img = torch.from_numpy(np.ascontiguousarray(so.make_batch(ocfg, 8, seed=5)[0])).cuda().view(8, 3, 32, 64)
    want = gm.infer_beam(img[::2].clone(), 3)
    room = torch.zeros(4, 3, 32, 80, dtype=torch.int8, device="cuda")
    room[..., :64] = img[::2]
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    for view in (img[::2], room[..., :64], img[::2].reshape(4, -1)):
        assert all(torch.equal(a, b) for a, b in zip(gm.infer_beam(view, 3), want))
        torch.cuda.synchronize()
        got = gm.infer_beam(view, 3, stream=st.cuda_stream)
        st.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_growth_while_another_stream_captures(lib, cuda):
    """The default stream's call that allocates meanwhile leaves the capture as it was."""
    import torch
    ocfg, _, gm = _pair(dict(img_w=64, max_len=4), 4, seed=78, train_steps=0)
    img = torch.from_numpy(np.ascontiguousarray(so.make_batch(ocfg, 4, seed=5)[0])).cuda()
    seq = torch.empty(4, 3, ocfg.steps, dtype=torch.int32, device="cuda")
    lengths, x = torch.empty(4, 3, dtype=torch.int32, device="cuda"), torch.ones(8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        y = x + 1
        rc = lib.trba_model_infer_beam(gm.h, img.data_ptr(), 4, 3, seq.data_ptr(), lengths.data_ptr(), None, None)
        y = y * 2
    assert rc == 0 and lib.trba_last_error() == 0
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 4).all()
    want = gm.infer_beam(img, 3)
    assert torch.equal(want[0], seq) and torch.equal(want[1], lengths)
