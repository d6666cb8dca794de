"""Beam-search operators (include/trba_decode.h, trba_b200.decode): against
the f64 oracle (oracle/decode_oracle.py), their refusals, and their use
together, captured into a graph and on other streams."""
import ctypes as C
import sys

import numpy as np
import pytest
import torch

from conftest import REPO

sys.path.insert(0, str(REPO / "oracle"))
import decode_oracle as do  # noqa: E402

from trba_b200 import decode  # noqa: E402

NEG = float("-inf")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------- oracle (CPU) --
def test_oracle_step_by_hand():
    lp = np.log(np.array([[0.5, 0.3, 0.2], [0.6, 0.3, 0.1]]))
    s, t, p, f = do.beam_select(lp[None], np.array([[-1.0, -1.1]], np.float32), None, eos=2)
    assert p.tolist() == [[1, 0]] and t.tolist() == [[0, 0]] and not f.any()
    assert np.allclose(s, [[np.float32(-1.1) + np.log(0.6), -1.0 + np.log(0.5)]])
    s, t, p, f = do.beam_select(lp[None], np.array([[-1.0, NEG]], np.float32), np.array([[True, False]]), eos=2)
    assert t.tolist() == [[2, 2]] and p.tolist() == [[0, 1]] and f.all() and s[0, 0] == -1.0 and s[0, 1] == NEG


def test_oracle_sequences_by_hand():
    tokens = np.array([[[5, 6]], [[7, 2]], [[2, 8]]])
    parents = np.array([[[0, 1]], [[1, 0]], [[1, 0]]])
    seq, n = do.beam_sequences(tokens, parents, eos=2, pad=-1)
    assert seq.tolist() == [[[5, -1, -1], [6, 7, 8]]] and n.tolist() == [[1, 3]]


# ----------------------------------------------------------- refusals (CPU) --
def _refused(lib, rc, word):
    assert rc == -1 and word in lib.trba_last_error_string(), (rc, lib.trba_last_error_string())
    lib.trba_clear_error()


def test_c_refusals(lib):
    lib.trba_clear_error()
    sel = lambda dtype=0, ld=10, lines=1, beams=2, vocab=10, eos=1, fin=None, p=None: lib.trba_beam_select(  # noqa: E731
        p, dtype, ld, p, fin, lines, beams, vocab, eos, p, p, p, p, None, 0, None)
    for kw in (dict(beams=0), dict(beams=33), dict(lines=-1), dict(vocab=0), dict(ld=9), dict(beams=32, vocab=1 << 27, ld=1 << 27)):
        _refused(lib, sel(**kw), b"bad sizes")
    _refused(lib, sel(eos=10), b"eos outside")
    _refused(lib, sel(eos=-2), b"eos outside")
    _refused(lib, sel(eos=-1, fin=C.c_void_p(64)), b"without an end token")
    _refused(lib, sel(dtype=3), b"element type")
    _refused(lib, sel(), b"null pointer")
    _refused(lib, sel(p=C.c_void_p(66)), b"not aligned")
    assert sel(lines=0) == 0
    _refused(lib, sel(vocab=1 << 16, ld=1 << 16, p=C.c_void_p(64)), b"workspace")
    assert lib.trba_beam_select_workspace(0, 1, 2, 10) == 0 < lib.trba_beam_select_workspace(0, 1, 2, 1 << 16)
    assert lib.trba_beam_select_workspace(0, 0, 2, 1 << 16) == 0 == lib.trba_beam_select_workspace(3, 1, 2, 1 << 16)
    one = (C.c_int64 * 11)(64, 64, -1, 8, 8, 1, 0, 0, 1, 0, 0)
    par = C.c_void_p(64)
    _refused(lib, lib.trba_beam_reorder(one, 1, par, 1, 2, None), b"negative")
    _refused(lib, lib.trba_beam_reorder((C.c_int64 * 11)(0, 64, 8, 8, 8, 1, 0, 0, 1, 0, 0), 1, par, 1, 2, None),
             b"null state")
    _refused(lib, lib.trba_beam_reorder(one, 1, None, 1, 2, None), b"null pointer")
    _refused(lib, lib.trba_beam_reorder(one, 1, par, 1, 33, None), b"bad sizes")
    _refused(lib, lib.trba_beam_reorder(one, -1, par, 1, 2, None), b"bad sizes")
    assert lib.trba_beam_reorder(None, 0, None, 1, 2, None) == 0
    assert lib.trba_beam_reorder((C.c_int64 * 11)(0, 0, 0, 8, 8, 1, 0, 0, 1, 0, 0), 1, par, 1, 2, None) == 0
    _refused(lib, lib.trba_beam_sequences(None, None, 3, 1, 2, 0, 0, None, None, None), b"null pointer")
    _refused(lib, lib.trba_beam_sequences(par, par, -1, 1, 2, 0, 0, par, par, None), b"bad sizes")
    _refused(lib, lib.trba_beam_sequences(par, par, 3, 1, 33, 0, 0, par, par, None), b"bad sizes")
    assert lib.trba_beam_sequences(None, None, 3, 0, 2, 0, 0, None, None, None) == 0
    assert lib.trba_last_error() == 0


def test_python_refusals():
    x, s = torch.zeros(6, 10), torch.zeros(2, 3)
    good = dict(logits=x, scores=s)

    def refused(exc, word, **kw):
        with pytest.raises(exc, match=word):
            decode.beam_select(**{**good, **kw})

    refused(ValueError, "CUDA")
    refused(TypeError, "torch tensor", logits=x.numpy())
    refused(TypeError, "float32, bfloat16", logits=x.double())
    refused(ValueError, "float32 tensor", scores=s.double())
    refused(ValueError, "do not fit", logits=x[:5])
    refused(ValueError, "do not fit", logits=x.view(3, 2, 10))
    refused(ValueError, "one stride", logits=torch.zeros(4, 3, 10)[::2])
    refused(ValueError, "contiguous", logits=torch.zeros(10, 6).T)
    refused(ValueError, "overlap", logits=torch.zeros(1, 10).expand(6, 10))
    refused(ValueError, "eos", eos=10)
    refused(ValueError, "end token", finished=torch.zeros(2, 3, dtype=torch.bool))
    refused(ValueError, "bool or uint8", finished=torch.zeros(2, 3), eos=1)
    refused(ValueError, "beams", logits=torch.zeros(33, 4), scores=torch.zeros(1, 33))
    p, t = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 4)
    for exc, word, args, kw in (
            (ValueError, "CUDA", ([t], p), {}), (ValueError, "int32", ([t], p.long()), {}),
            (ValueError, "expected lines", ([t[:5]], p), {}), (ValueError, "no dimension", ([t], p), dict(dim=2)),
            (ValueError, "out has", ([t], p), dict(out=[])), (ValueError, "shape and type", ([t], p), dict(out=[t.double()])),
            (ValueError, "overlaps", ([t], p), dict(out=[t])), (ValueError, "broadcast", ([t], p), dict(out=[torch.zeros(6, 1).expand(6, 4)])),
            (TypeError, "torch tensor", ([t.numpy()], p), {})):
        with pytest.raises(exc, match=word):
            decode.beam_reorder(*args, **kw)
    k = torch.zeros(4, 2, 3, dtype=torch.int32)
    for exc, word, args, kw in ((ValueError, "CUDA", (k, k), {}), (ValueError, "int32", (k, k.long()), {}),
                                (ValueError, "int32", (k, k[:3]), {}), (ValueError, "32 bits", (k, k), dict(eos=1 << 31))):
        with pytest.raises(exc, match=word):
            decode.beam_sequences(*args, **kw)


def test_state_views():
    """The views that beam_reorder makes of strided states (bytes)."""
    cache = torch.zeros(6, 4, 10, 8, dtype=torch.float16)
    got = decode._state(cache[:, :, :7], torch.zeros(6, 4, 7, 8, dtype=torch.float16), 0)
    assert got[2:] == (7 * 16, 4 * 160, 4 * 112, 4, 160, 112, 1, 0, 0)
    layers = torch.zeros(3, 6, 5)
    assert decode._state(layers, layers.clone(), 1)[2:] == (20, 20, 20, 1, 0, 0, 3, 120, 120)
    assert decode._state(torch.zeros(6), torch.zeros(6), 0)[2:] == (4, 4, 4, 1, 0, 0, 1, 0, 0)
    assert decode._state(torch.zeros(4, 6).T, torch.zeros(6, 4), 0)[2:] == (4, 4, 16, 4, 24, 4, 1, 0, 0)
    with pytest.raises(ValueError, match="contiguous"):
        decode._state(torch.zeros(6, 4, 8, 6)[:, :, :5, ::2], torch.zeros(6, 4, 5, 3), 0)


def test_too_many_states_are_refused_before_any_is_moved(lib):
    """A state of too many parts behind a launch's worth of others."""
    lib.trba_clear_error()
    good, bad = (64, 1 << 20, 16, 16, 16, 1, 0, 0, 1, 0, 0), (64, 1 << 30, 1, 1 << 24, 1 << 23, 1 << 24, 2, 1, 1, 0, 0)
    launches = lib.trba_launch_count()
    for n, state in ((0, bad), (16, bad), (20, bad), (16, (64, 64, -1, 8, 8, 1, 0, 0, 1, 0, 0))):
        views = (C.c_int64 * (11 * (n + 1)))(*good * n, *state)
        assert lib.trba_beam_reorder(views, n + 1, C.c_void_p(64), 256, 1, None) == -1
        assert lib.trba_launch_count() == launches
        lib.trba_clear_error()
    big, half = (torch.empty(256, n, dtype=torch.int8, device="meta") for n in (1 << 24, 1 << 23))
    with pytest.raises(ValueError, match="too large"):
        decode._state(big[:, ::2], half, 0)
    assert decode._state(big[:, ::2][:100], half[:100], 0)[5] == 1 << 23
    assert decode._state(big, big, 0)[2] == 1 << 24


def test_outputs_that_share_memory():
    """The rule that outputs are checked by, on the host."""
    m = torch.zeros(60)
    apart = lambda w, r=(), same=(): decode._check_apart({f"w{i}": t for i, t in enumerate(w)}, {f"r{i}": t for i, t in enumerate(r)}, same)  # noqa: E731
    apart([m[:10], m[10:20]], [m[20:], m[20:]])  # inputs may be anything
    apart([m[:0], m[5:5]], [m])
    apart([m[:10]], [m[:10]], {("w0", "r0")})
    apart([m[:40].view(4, 10)[:, :5]], [m[40:]])
    for w, r, word in (([m[:10], m[9:20]], [], "w0 overlaps w1"), ([m[30:], m[:31]], [], "overlaps"), ([m[:10]], [m[:10]], "w0 overlaps r0"),
                       ([m[:10]], [m], "w0 overlaps r0"), ([m], [m[7:8]], "w0 overlaps r0"), ([m[:1].expand(4)], [], "broadcast"),
                       ([m.as_strided((4, 5), (4, 1))], [], "itself"), ([m.as_strided((5, 5), (1, 1))], [], "itself")):
        with pytest.raises(ValueError, match=word):
            apart(w, r)
    for w, r in (([m[:10]], [m[:11]]), ([m[:10]], [m[1:11]])):
        with pytest.raises(ValueError, match="overlaps"):
            apart(w, r, {("w0", "r0")})
    p, t = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 4)
    o = torch.zeros(6, 4)
    for states, out in (([t, t], [o, o]), ([t[:, :2], t], [o[:, 2:], o])):
        with pytest.raises(ValueError, match="overlaps"):
            decode.beam_reorder(states, p, out=out)
    with pytest.raises(ValueError, match="overlaps parents"):
        decode.beam_reorder([torch.zeros(6, 1, dtype=torch.int32)], p, out=[p.view(6, 1)])


def test_streams_are_torchs():
    for stream in (0, C.c_void_p(64), "0"):
        with pytest.raises(TypeError, match="torch.cuda.Stream"):
            decode._on(torch.device("cuda", 0), stream)


def test_interleaved_tensors():
    """Side by side in a wider row, or not: by the addresses of all elements."""
    def bytes_of(t):
        at = np.zeros((), np.int64)
        for n, st in zip(t.shape, t.stride()):
            at = at[..., None] + np.arange(n) * st * t.element_size()
        return set((at.ravel()[:, None] + t.data_ptr() + np.arange(t.element_size())).ravel().tolist())

    rng = np.random.default_rng(0)
    base = torch.zeros(4000, dtype=torch.uint8)
    seen = [0, 0]
    for _ in range(3000):
        ts = []
        for _ in range(2):
            dtype = (torch.uint8, torch.int16, torch.int32)[rng.integers(3)]
            size = torch.empty(0, dtype=dtype).element_size()
            strides = [int(st) for st in rng.choice([1, 2, 8, 12, 24, 48, 96], 3)]
            shape = [int(n) for n in rng.integers(1, 5, 3)]
            ts.append(base.view(dtype).as_strided(shape, strides, int(rng.integers(60 // size))))
        share = bool(bytes_of(ts[0]) & bytes_of(ts[1]))
        assert not (decode._interleaved(*ts) and share)
        assert decode._interleaved(*ts) == decode._interleaved(*ts[::-1])
        seen[decode._interleaved(*ts)] += not share
    assert min(seen) > 50
    w = torch.zeros(6, 2, 8)
    assert decode._interleaved(w[:, 0], w[:, 1]) and not decode._interleaved(w[:, 0], w[:, 0])
    assert decode._interleaved(w[:, 0, :5], w[:, 1]) and not decode._interleaved(w[:, 0], w.view(6, 16)[:, 7:])
    assert decode._interleaved(w[:, 0], w.view(96)[88:].view(1, 8)) is False  # (no stride in common; their ranges decide)


# --------------------------------------------------------------- GPU: select --
# A score is off by at most: half a step of f32 (2^-24 of it); the f32
# exponentials, whose relative error is 2^-22 (the function) + 2^-23 |t| (t
# and t * log2(e) rounded), weighted with the probabilities: E|t| <= log V + 1
# < 13 below 2^17 tokens, so 2^-22 + 13 * 2^-23 < 2^-19 on the logarithm.
def tol(scores):
    return 2.0 ** -19 + 2.0 ** -24 * np.where(np.isfinite(scores), np.abs(scores), 0)


def check_step(step, logits, scores, finished, eos):
    """Scores within their tolerance, and every choice one that the oracle
    makes: equal to it, or within twice the tolerance of it in f64."""
    x = logits.float().cpu().numpy().reshape(*scores.shape, -1)
    s, f = scores.cpu().numpy(), None if finished is None else finished.cpu().numpy().astype(bool)
    want = do.beam_select(x, s, f, eos)
    got = [t.cpu().numpy() for t in step]
    tot = do.totals(x, s, f, eos)
    L, K, V = tot.shape
    assert np.array_equal(np.isfinite(got[0]), np.isfinite(want[0]))
    live = np.isfinite(want[0])
    assert (np.abs(got[0][live] - want[0][live]) <= tol(want[0][live])).all()
    for k in range(1, 4):
        assert np.array_equal(got[k][~live], want[k][~live])
    ll, kk = np.nonzero(live)
    chosen = tot[ll, got[2][ll, kk], got[1][ll, kk]]
    assert (np.abs(chosen - want[0][ll, kk]) <= 2 * tol(want[0][ll, kk])).all()
    flat = got[2].astype(np.int64) * V + got[1]
    for b in range(L):
        assert len(set(flat[b][live[b]])) == live[b].sum()
    fin = (got[1] == eos) | (np.take_along_axis(f, got[2], 1) if f is not None else False)
    assert np.array_equal(got[3][live], fin[live] if eos >= 0 else np.zeros(live.sum(), bool))
    return got, want


def make(L, K, V, dtype, seed, dev="cuda", mask=0.0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(L * K, V, generator=g) * scale
    if mask:
        x[torch.rand(L * K, V, generator=g) < mask] = NEG
    s = -torch.randn(L, K, generator=g).abs().cumsum(1)
    f = torch.rand(L, K, generator=g) < 0.2
    return x.to(DTYPES[dtype]).to(dev), s.to(dev), f.to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("L,K,V", [(1, 1, 1), (1, 1, 130), (1, 5, 130), (3, 32, 2), (2, 7, 31), (2, 8, 33), (5, 3, 255),
                                   (130, 5, 130), (2, 32, 1000), (1, 16, 5003), (7, 4, 4096), (1, 1, 70001),
                                   (3, 10, 20000), (40, 6, 2049)])
def test_select_matches_oracle(L, K, V, dtype, lib, cuda):
    for seed, (mask, first) in enumerate([(0.0, False), (0.7, False), (0.0, True)]):
        x, s, f = make(L, K, V, dtype, seed + 10 * L, mask=mask)
        if first:
            s[:, 1:] = NEG
            f = None
        eos = min(2, V - 1)
        check_step(decode.beam_select(x, s, f, eos=eos), x, s, f, eos)
    check_step(decode.beam_select(x, s, eos=-1), x, s, None, -1)
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [37, 130, 3001, 40000])
def test_select_ties_go_to_the_lowest_index(V, dtype, cuda):
    """Equal logits, within a row and across rows whose starts are aligned differently."""
    K = 6
    x = torch.zeros(2 * K, V, dtype=DTYPES[dtype], device="cuda")
    x[K:, ::3] = 1.5  # line 1: every third token ties at the top
    s = torch.full((2, K), -1.0, device="cuda")
    step = decode.beam_select(x, s)
    assert step.parents.tolist() == [[0] * K] * 2
    assert step.tokens[0].tolist() == list(range(K)) and step.tokens[1].tolist() == [3 * k for k in range(K)]
    # one value, many beams with one candidate each: rows are equal, beams tie
    y = torch.full((K, V), NEG, dtype=DTYPES[dtype], device="cuda")
    y[:, V - 1] = -2.0
    step = decode.beam_select(y, s[:1])
    assert step.parents.tolist() == [list(range(K))] and step.tokens.tolist() == [[V - 1] * K]
    g = torch.Generator().manual_seed(V)
    row = (torch.randn(V, generator=g) * 3).to(DTYPES[dtype]).cuda()
    step = decode.beam_select(row.expand(K, V).contiguous(), s[:1])
    best = (row == row.max()).nonzero().flatten().tolist()  # equal rows: each beam's best tokens, beam by beam
    want = [(k, v) for k in range(K) for v in best][:K]
    assert step.parents.tolist() == [[k for k, _ in want]] and step.tokens.tolist() == [[v for _, v in want]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("order", ["up", "down", "saw"])
def test_select_sorted_rows(order, dtype, cuda):
    """Ascending rows replace the best at every element."""
    V, K = 9001, 9
    r = torch.linspace(-30, 30, V)
    x = {"up": r, "down": r.flip(0), "saw": r.view(-1)[torch.arange(V).mul(37).remainder(V)]}[order].to(DTYPES[dtype])
    x = x.expand(K, V).contiguous().cuda()
    s = -torch.arange(K, device="cuda", dtype=torch.float32)[None] * 1e-3
    check_step(decode.beam_select(x, s, eos=0), x, s, None, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [515, 9001, 70000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_special_values(dtype, V, cuda):
    t = DTYPES[dtype]
    low = torch.finfo(t).min
    K = 4
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(8 * K, V, generator=g) * 2).to(t)
    v = x.view(8, K, V)
    v[0] = NEG                       # nothing left on the line
    v[1, :, 1:] = NEG                # one token a row
    v[2] = low                       # a row of the type's lowest value is uniform
    v[3, :, :-2] = low               # two tokens far above a mask of the lowest value
    v[4, :, ::2] = float("nan")      # NaN counts as -inf
    v[5, 0, [7, 300]] = float("inf")  # two tokens share the row
    v[6] = float("nan")
    v[7, :2] = NEG                   # two of the line's rows are empty
    s = -torch.arange(8 * K, dtype=torch.float32).view(8, K) * 0.25
    s[4, 1] = float("nan")
    s[7, 3] = NEG
    x, s = x.cuda(), s.cuda()
    got, _ = check_step(decode.beam_select(x, s, eos=5), x, s, None, 5)
    assert (got[0][0] == NEG).all() and got[1][0].tolist() == [5] * K and got[2][0].tolist() == [0, 1, 2, 3] and got[3][0].all()
    assert (got[0][6] == NEG).all()
    fin = torch.ones(8, K, dtype=torch.uint8, device="cuda")  # all finished: logits do not matter
    got, _ = check_step(decode.beam_select(x, s, fin, eos=5), x, s, fin, 5)
    assert (got[1] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("off,ld", [(0, 301), (1, 304), (3, 303), (4, 320), (7, 309)])
def test_select_strides_and_offsets(off, ld, dtype, cuda):
    L, K, V = 3, 5, 300
    buf = torch.full((L * K * ld + off + 8,), 60000.0, device="cuda").to(DTYPES[dtype])
    x, s, f = make(L, K, V, dtype, off + ld)
    view = buf[off:off + L * K * ld].view(L * K, ld)[:, :V]
    view.copy_(x)
    check_step(decode.beam_select(view, s, f, eos=2), x, s, f, 2)
    check_step(decode.beam_select(view.unflatten(0, (L, K)), s.T.contiguous().T, f, eos=2), x, s, f, 2)
    one = view[::K][:, None]  # one beam a line, every K-th row
    check_step(decode.beam_select(one, s[:, :1], f[:, :1], eos=2), x[::K], s[:, :1], f[:, :1], 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_long_rows_at_odd_addresses(dtype, cuda):
    """Rows of many segments whose starts miss 16-byte boundaries in every way."""
    L, K, V = 2, 4, 20011
    buf = torch.full((L * K * (V + 2) + 16,), 60000.0, device="cuda").to(DTYPES[dtype])
    for off in range(8):
        x, s, f = make(L, K, V, dtype, off)
        view = buf[off:off + L * K * (V + 1)].view(L * K, V + 1)[:, :V]
        view.copy_(x)
        check_step(decode.beam_select(view, s, f, eos=2), x, s, f, 2)


@pytest.mark.gpu
def test_select_in_place_and_repeatable(lib, cuda):
    x, s, f = make(9, 6, 7001, "bf16", 5)
    a = decode.beam_select(x, s, f, eos=2)
    b = decode.beam_select(x, s, f, eos=2)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    s2, f2 = s.clone(), f.clone()
    c = decode.beam_select(x, s2, f2, eos=2, out=decode.BeamStep(s2, torch.empty_like(a.tokens),
                                                              torch.empty_like(a.parents), f2))
    assert c.scores is s2 and all(torch.equal(p, q) for p, q in zip(a, c))
    for bad in (a._replace(scores=s[:, :5]), a._replace(finished=f.to(torch.uint8)), a._replace(tokens=a.tokens.long())):
        with pytest.raises(ValueError, match="out."):
            decode.beam_select(x, s, f, eos=2, out=bad)
    empty = decode.beam_select(x[:0], s[:0], f[:0], eos=2)
    assert empty.scores.shape == (0, 6)
    assert lib.trba_last_error() == 0


# -------------------------------------------------------------- GPU: reorder --
def rows_of(parents):
    L, K = parents.shape
    return (torch.arange(L, device=parents.device)[:, None] * K + parents).reshape(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8, torch.int64, torch.bool, torch.complex128])
@pytest.mark.parametrize("L,K,W", [(1, 1, 1), (1, 5, 64), (3, 4, 255), (200, 5, 17), (2, 32, 4099), (1, 2, 100003)])
def test_reorder_matches_indexing(L, K, W, dtype, lib, cuda):
    g = torch.Generator(device="cuda").manual_seed(W)
    par = torch.randint(0, K, (L, K), generator=g, device="cuda", dtype=torch.int32)
    a = torch.randint(0, 120, (L * K, W), generator=g, device="cuda").to(dtype)
    b = torch.randint(0, 120, (3, L * K, 2, W), generator=g, device="cuda").to(dtype)
    rows = rows_of(par)
    assert torch.equal(decode.beam_reorder([a], par)[0], a[rows])
    assert torch.equal(decode.beam_reorder([b], par, dim=1)[0], b[:, rows])
    assert torch.equal(decode.beam_reorder([b], par, dim=-3)[0], b[:, rows])
    if W > 2:  # views that start at odd places and skip
        assert torch.equal(decode.beam_reorder([a[:, 1:-1]], par)[0], a[rows][:, 1:-1])
        assert torch.equal(decode.beam_reorder([b[0, :, :, 1:]], par)[0], b[0][rows][:, :, 1:])
        assert torch.equal(decode.beam_reorder([b[::2]], par, dim=1)[0], b[::2][:, rows])
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
def test_reorder_many_states_and_outputs(cuda):
    g = torch.Generator(device="cuda").manual_seed(2)
    L, K = 6, 5
    par = torch.randint(0, K, (L, K), generator=g, device="cuda", dtype=torch.int32)
    rows = rows_of(par)
    cache = [torch.randn(L * K, 4, 20, 8 + i, generator=g, device="cuda").bfloat16() for i in range(37)]
    part = [c[:, :, :11] for c in cache]
    out = [torch.full_like(c, 7.0) for c in cache]
    got = decode.beam_reorder(part, par, out=[o[:, :, :11] for o in out])
    for c, o, x in zip(cache, out, got):
        assert x.data_ptr() == o.data_ptr() and torch.equal(o[:, :, :11], c[rows][:, :, :11])
        assert (o[:, :, 11:] == 7).all()  # the rest of the room is left as it was
    assert decode.beam_reorder([], par) == []
    assert decode.beam_reorder([torch.empty(30, 0, device="cuda")], par)[0].shape == (30, 0)
    none = decode.beam_reorder([torch.empty(0, 3, device="cuda")], par[:0])[0]
    assert none.shape == (0, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,W", [(torch.float32, 8), (torch.int8, 3), (torch.bfloat16, 255)])
def test_reorder_between_halves_of_one_buffer(dtype, W, cuda):
    """Two sets of states in one allocation, used in turn."""
    par = torch.tensor([[2, 0, 2], [1, 1, 0]], dtype=torch.int32, device="cuda")
    both = torch.randint(0, 100, (6, 2, W), device="cuda").to(dtype)
    want, layers = both[:, 0][rows_of(par)], torch.randint(0, 100, (4, 2, 6, W), device="cuda").to(dtype)
    keep, want_l = both[:, 0].clone(), layers[:, 1][:, rows_of(par)]
    decode.beam_reorder([both[:, 0]], par, out=[both[:, 1]])
    assert torch.equal(both[:, 1], want) and torch.equal(both[:, 0], keep)
    decode.beam_reorder([layers[:, 1]], par, dim=1, out=[layers[:, 0]])
    assert torch.equal(layers[:, 0], want_l)


@pytest.mark.gpu
def test_reorder_leaves_rows_of_bad_parents(cuda):
    a = torch.arange(40.0, device="cuda").view(8, 5)
    par = torch.tensor([[0, -1, 3, 4], [1 << 30, 2, -(1 << 31), 1]], dtype=torch.int32, device="cuda")
    out = torch.full_like(a, -5.0)
    decode.beam_reorder([a], par, out=[out])
    for r, src in enumerate([0, None, 3, None, None, 6, None, 5]):
        assert torch.equal(out[r], a[src] if src is not None else torch.full_like(a[0], -5.0)), r


@pytest.mark.gpu
def test_reorder_offsets_past_32_bits(cuda):
    """Rows of a cache whose byte offsets pass 2^32 (5 GB of room, little of it copied)."""
    rows, row = 5, 1 << 30
    cache = torch.empty(rows, row, dtype=torch.int8, device="cuda")
    for r in range(rows):
        cache[r, :100].fill_(r + 1)
        cache[r, -100:].fill_(-r - 1)
    par = torch.tensor([[4, 3, 2, 1, 0]], dtype=torch.int32, device="cuda")
    head, tail = decode.beam_reorder([cache[:, :100], cache[:, -100:]], par)
    assert head[:, 0].tolist() == [5, 4, 3, 2, 1] and tail[:, 99].tolist() == [-5, -4, -3, -2, -1]


# ------------------------------------------------------------ GPU: sequences --
@pytest.mark.gpu
@pytest.mark.parametrize("T,L,K", [(0, 2, 3), (1, 1, 1), (1, 3, 32), (2, 2, 2), (21, 130, 5), (31, 1, 7), (64, 3, 32),
                                   (65, 2, 16), (500, 3, 1), (1001, 2, 9), (2500, 1, 32)])
def test_sequences_match_oracle(T, L, K, lib, cuda):
    rng = np.random.default_rng(T + K)
    tok = rng.integers(3, 60, (T, L, K)).astype(np.int32)
    tok[rng.random((T, L, K)) < 1.0 / (T + 1)] = 2
    par = rng.integers(0, K, (T, L, K)).astype(np.int32)
    if T:
        par[0] = -7  # not used
    t, p = torch.from_numpy(tok).cuda(), torch.from_numpy(par).cuda()
    for eos, pad in ((2, 0), (-1, 9)):
        want = do.beam_sequences(tok, np.where(np.arange(T)[:, None, None] == 0, 0, par), eos, pad)
        got = decode.beam_sequences(t, p, eos=eos, pad=pad)
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("K", [5, 8])
@pytest.mark.parametrize("T", [3, 40, 700])
def test_sequences_with_bad_parents(T, K, cuda):
    rng = np.random.default_rng(T)
    L = 4
    tok = rng.integers(3, 60, (T, L, K)).astype(np.int32)
    par = rng.integers(0, K, (T, L, K)).astype(np.int32)
    par[0] = -1
    par[T - 1, 0, 1] = K
    par[1, 1] = -3
    par[T // 2, 2, 2] = 1 << 30
    ref = par.copy()
    ref[0] = 0
    want = do.beam_sequences(tok, ref, 2, 0)
    got = decode.beam_sequences(torch.from_numpy(tok).cuda(), torch.from_numpy(par).cuda(), eos=2)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
    assert (want[1][1] == -1).all() and want[1][0, 1] == -1 and (want[1][3] == T).all()


# ------------------------------------------------------------- GPU: together --
def toy_decoder(L, K, V, H, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    emb, w = torch.randn(V, H, generator=g, device="cuda"), torch.randn(H, V, generator=g, device="cuda") * 0.7

    def step(h, tokens):
        h = torch.tanh(0.5 * h + emb[tokens.reshape(-1).long()])
        return h, (h @ w).to(dtype)

    return step


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 4, 12])
def test_beam_search_run(K, cuda):
    """A whole search, step by step against the oracle on the same logits, and
    its sequences against a search that carries the token lists along."""
    L, V, H, T, eos = 5, 61, 16, 12, 2
    decoder = toy_decoder(L, K, V, H, K)
    h = torch.zeros(L * K, H, device="cuda")
    scores = torch.full((L, K), NEG, device="cuda")
    scores[:, 0] = 0
    fin = torch.zeros(L, K, dtype=torch.bool, device="cuda")
    tokens = torch.ones(L, K, dtype=torch.int32, device="cuda")
    paths = [[[] for _ in range(K)] for _ in range(L)]
    hist = []
    for _ in range(T):
        h, logits = decoder(h, tokens)
        step = decode.beam_select(logits, scores, fin, eos=eos)
        check_step(step, logits, scores, fin, eos)
        h = decode.beam_reorder([h], step.parents)[0]
        scores, tokens, parents, fin = step
        hist.append((tokens, parents))
        t, p = tokens.tolist(), parents.tolist()
        paths = [[paths[b][p[b][k]] + [t[b][k]] for k in range(K)] for b in range(L)]
    seq, n = decode.beam_sequences(torch.stack([t for t, _ in hist]), torch.stack([p for _, p in hist]), eos=eos, pad=-1)
    for b in range(L):
        for k in range(K):
            path = paths[b][k]
            cut = path.index(eos) if eos in path else T
            assert seq[b, k].tolist() == path[:cut] + [-1] * (T - cut) and n[b, k] == cut
    assert (scores[:, :-1] >= scores[:, 1:]).all()


@pytest.mark.gpu
def test_captured_and_on_other_streams(lib, cuda):
    """The step captured into two graphs that run at once, replayed on new inputs, and on a stream given by hand."""
    L, K, V, H = 7, 5, 1003, 40
    inputs = [make(L, K, V, "bf16", 50 + i) for i in range(4)]
    hs = [torch.randn(L * K, H, device="cuda") for _ in range(4)]

    def once(x, s, f, h, stream=None):
        st = decode.beam_select(x, s, f, eos=2, stream=stream)
        h2 = decode.beam_reorder([h], st.parents, stream=stream)[0]
        return (*st, h2, *decode.beam_sequences(st.tokens[None], st.parents[None], eos=2, stream=stream))

    want = [once(*i, h) for i, h in zip(inputs, hs)]
    graphs = []
    for q in range(2):
        buf = [t.clone() for t in (*inputs[q], hs[q])]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = once(*buf)
        graphs.append((g, buf, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for r in range(2):
        for q, (g, buf, out) in enumerate(graphs):
            with torch.cuda.stream(streams[q]):
                for b, t in zip(buf, (*inputs[2 * r + q], hs[2 * r + q])):
                    b.copy_(t)
                g.replay()
        torch.cuda.synchronize()
        for q, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[2 * r + q]))
    got = once(*inputs[0], hs[0], stream=streams[0])
    streams[0].synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
def test_overlapping_outputs_are_refused(cuda):
    x, s, f = make(3, 4, 50, "f32", 1)
    new = decode.beam_select(x, s, f, eos=2)
    room = torch.zeros(24, device="cuda")
    bad = [new._replace(parents=new.tokens), new._replace(tokens=s.view(torch.int32)), new._replace(scores=x.view(-1)[6:18].view(3, 4)),
           new._replace(tokens=new.scores.view(torch.int32)), new._replace(finished=room.view(torch.bool)[:12].view(3, 4), scores=room[1:13].view(3, 4))]
    for out in bad:
        with pytest.raises(ValueError, match="overlaps"):
            decode.beam_select(x, s, f, eos=2, out=out)
    shifted = room[4:16].view(3, 4).copy_(s)  # the scores one line further down in one buffer
    with pytest.raises(ValueError, match="out.scores overlaps scores"):
        decode.beam_select(x, shifted, f, eos=2, out=new._replace(scores=room[:12].view(3, 4)))
    tok, par = torch.zeros(2, 5, 3, 4, dtype=torch.int32, device="cuda").unbind()
    seq, n = decode.beam_sequences(tok, par)
    for out in ((tok.view(3, 4, 5), n), (seq, seq.view(-1)[:12].view(3, 4)), (seq, par.view(-1)[:12].view(3, 4))):
        with pytest.raises(ValueError, match="overlaps"):
            decode.beam_sequences(tok, par, out=out)
    decode.beam_select(x, s, f, eos=2, out=decode.BeamStep(s, tok[0], par[0], f))  # in place, into a history
    assert torch.equal(s, new.scores) and torch.equal(tok[0], new.tokens) and torch.equal(f, new.finished)


@pytest.mark.gpu
def test_negated_and_conjugated_views(cuda):
    """torch's lazy views are read as the values they stand for."""
    par = torch.tensor([[1, 1, 0]], dtype=torch.int32, device="cuda")
    z = torch.randn(3, 5, dtype=torch.complex64, device="cuda")
    neg = torch._neg_view(torch.randn(3, 5, device="cuda"))
    assert z.conj().is_conj() and neg.is_neg()
    got = decode.beam_reorder([z.conj(), neg, z.conj().imag, torch._neg_view(z.conj())], par)
    for g, t in zip(got, (z.conj(), neg, z.conj().imag, -z.conj())):
        assert torch.equal(g.resolve_conj().resolve_neg(), t.resolve_conj().resolve_neg()[par[0].long()])
    for t, o in ((z, z.clone().conj()), (neg, torch._neg_view(torch.zeros(3, 5, device="cuda")))):
        with pytest.raises(ValueError, match="view"):
            decode.beam_reorder([t], par, out=[o])
    x, s, f = make(2, 3, 70, "f32", 4)
    want = decode.beam_select(x, s, f, eos=2)
    got = decode.beam_select(torch._neg_view(-x), torch._neg_view(-s), f, eos=2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = torch.full((6, 80), 1e4, device="cuda")
    wide[:, :70] = -x
    got = decode.beam_select(torch._neg_view(wide[:, :70]), s, f, eos=2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="out.scores"):
        decode.beam_select(x, s, f, eos=2, out=want._replace(scores=torch._neg_view(s.clone())))
    t, p = (torch.randint(0, 3, (4, 2, 3), dtype=torch.int32, device="cuda") for _ in range(2))
    got, want = decode.beam_sequences(torch._neg_view(-t), torch._neg_view(-p)), decode.beam_sequences(t, p)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,L,K,V", [("f32", 1, 2, 1300003), ("bf16", 1, 1, 2300001), ("f16", 2, 1, 2100007)])
def test_select_rows_of_millions(dtype, L, K, V, cuda):
    """Segments of more batches than there are spans to remember: several
    batches a span are looked at again.  Scores as everywhere: E|t| <= log V +
    1 < 16 here, so 2^-22 + 16 * 2^-23 is still below 2^-18."""
    x, s, f = make(L, K, V + 3, dtype, V & 7, mask=0.3)
    for off in (0, 1, 3):
        view = x[:, off:off + V]
        got = [t.cpu().numpy() for t in decode.beam_select(view, s, eos=2)]
        rows = view.double().view(L, K, V)
        total = s.double()[:, :, None] + rows - torch.logsumexp(rows, -1, keepdim=True)
        best = torch.sort(total.view(L, K * V), dim=1, descending=True, stable=True)
        want, at = best[0][:, :K].cpu().numpy(), best[1][:, :K].cpu().numpy()
        tol18 = 2.0 ** -18 + 2.0 ** -24 * np.abs(want)
        assert (np.abs(got[0] - want) <= tol18).all()
        flat = got[2].astype(np.int64) * V + got[1]
        chosen = np.take_along_axis(total.view(L, K * V).cpu().numpy(), flat, 1)
        assert (np.abs(chosen - want) <= 2 * tol18).all() and all(len(set(r)) == K for r in flat.tolist())
        # within one beam the order is that of the logits, exactly: ties to the lowest token
        if K == 1:
            assert np.array_equal(flat, at)
    # a single largest element anywhere in a span of several batches, ties to the lowest
    y = torch.zeros(L * K, V, dtype=DTYPES[dtype], device="cuda")
    for at in (0, 511, 8191, 8192, 8704, 16383, 1050624, V // 2 + 1, V - 1):
        y.zero_()
        y[:, at] = 1.0
        y[:, V - 1] = 1.0
        step = decode.beam_select(y, torch.zeros(L, K, device="cuda"))
        want = [(k, v) for k in range(K) for v in sorted({at, V - 1})][:K]
        assert list(zip(step.parents[-1].tolist(), step.tokens[-1].tolist())) == want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_select_largest_vocabulary(dtype, lib, cuda):
    """2^30 tokens: zeros, a few of them higher.  |t| is at most 12 here, and a
    thread's partial sum takes 5 additions: 2^-22 + 12 * 2^-23 + 5 * 2^-24 < 2^-18."""
    tol = lambda s: 2.0 ** -18 + 2.0 ** -24 * abs(s)  # noqa: E731
    V = 1 << 30
    x = torch.zeros(1, V, dtype=DTYPES[dtype], device="cuda")
    s = torch.tensor([[-1.5]], device="cuda")
    step = decode.beam_select(x, s)
    assert step.tokens.item() == 0 and abs(step.scores.item() + 1.5 + np.log(V)) <= tol(22.3)
    for at in (V - 1, V // 2 + 12345, 777):  # each higher than the one before
        x[0, at] = x.max() + 4
        step = decode.beam_select(x, s, torch.zeros(1, 1, dtype=torch.bool, device="cuda"), eos=V - 1)
        n = int(round(x.max().item() / 4))
        want = -1.5 + 4 * n - np.log(V - n + sum(np.exp(4.0 * k) for k in range(1, n + 1)))
        assert step.tokens.item() == at and abs(step.scores.item() - want) <= tol(want)
        assert step.finished.item() == (at == V - 1)
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,K", [(300001, 2), (70000, 32)])
def test_sequences_of_many_steps(T, K, lib, cuda):
    """Many chunks of steps, the last first."""
    rng = np.random.default_rng(K)
    tok, par = rng.integers(3, 60, (T, 1, K)).astype(np.int32), rng.integers(0, K, (T, 1, K)).astype(np.int32)
    tok[T // 3 * 2] = 2
    par[0] = 0
    slot, path = np.arange(K), np.empty((T, K), np.int32)
    for t in range(T - 1, -1, -1):
        path[t] = tok[t, 0, slot]
        slot = par[t, 0, slot]
    seq, n = decode.beam_sequences(torch.from_numpy(tok).cuda(), torch.from_numpy(par).cuda(), eos=2, pad=-1)
    assert (n == T // 3 * 2).all()
    path[T // 3 * 2:] = -1
    assert np.array_equal(seq[0].cpu().numpy(), path.T)
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
def test_long_rows_captured(lib, cuda):
    """The two launches of long rows in two graphs that run at once, on new inputs."""
    L, K, V = 3, 5, 30011
    inputs = [make(L, K, V, "bf16", 70 + i) for i in range(4)]
    want = [decode.beam_select(*i, eos=2) for i in inputs]
    graphs = []
    for q in range(2):
        buf = [t.clone() for t in inputs[q]]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = decode.beam_select(*buf, eos=2)
            for _ in range(3):  # a step on the scores of the last, in one graph
                again = decode.beam_select(buf[0], out.scores, out.finished, eos=2)
        graphs.append((g, buf, out, again, torch.cuda.Stream()))
    for r in range(2):
        for q, (g, buf, _, _, st) in enumerate(graphs):
            with torch.cuda.stream(st):
                for b, t in zip(buf, inputs[2 * r + q]):
                    b.copy_(t)
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for q, (_, buf, out, again, _) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[2 * r + q]))
            check_step(again, buf[0], out.scores, out.finished, 2)
    assert lib.trba_last_error() == 0
