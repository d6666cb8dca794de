"""LinearInt4 (include/trba_ops.h, trba_b200.ops): the 4-bit linear layer
against its f64 oracle (oracle/decode_oracle.py), its quantisation, its
refusals, and a decoding loop that reads its weights through it."""
import ctypes as C
import sys

import numpy as np
import pytest
import torch

from conftest import REPO

sys.path.insert(0, str(REPO / "oracle"))
import decode_oracle as do  # noqa: E402

from trba_b200 import decode  # noqa: E402
from trba_b200.ops import LinearInt4  # noqa: E402

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------ oracle (CPU) --
def test_oracle_quantisation():
    w = np.array([[7.0, -7.0, 0.5, -0.5, 1.5, 0.49, 3.5], [0.0] * 7, [14.0, 1.0, -1.0, 3.0, -13.1, 0.0, 5.0]], np.float32)
    q, s = do.int4_quantize(w, 32)
    assert s.ravel().tolist() == [1.0, 1.0, 2.0] and q.shape == (3, 4)
    back = do.int4_weights(q, s, 7, 32)
    assert back.tolist() == [[7, -7, 1, -1, 2, 0, 4], [0] * 7, [14, 2, -2, 4, -14, 0, 6]]
    rng = np.random.default_rng(0)
    w = rng.standard_normal((5, 300)).astype(np.float32)
    q, s = do.int4_quantize(w, 128)
    assert s.shape == (5, 3)
    assert (np.abs(do.int4_weights(q, s, 300, 128) - w) <= 0.5001 * np.repeat(s, 128, 1)[:, :300]).all()


# ---------------------------------------------------------- refusals (CPU) --
def test_c_refusals(lib):
    lib.trba_clear_error()

    def refused(rc, word):
        assert rc in (-1, None, 0) and word in lib.trba_last_error_string(), lib.trba_last_error_string()
        assert rc != 0 or rc is None
        lib.trba_clear_error()

    p = C.c_void_p(64)
    for ins, outs, group in ((0, 4, 32), (4, 0, 32), (4, (1 << 30) + 1, 32), ((1 << 30) + 1, 4, 32), (4, 4, 0), (4, 4, 16), (4, 4, 48), (4, 4, 129), (4, 4, -32)):
        refused(lib.trba_linear_int4_create(ins, outs, group, p, None), b"bad arguments")
        refused(lib.trba_linear_int4_create_codes(ins, outs, group, p, 1 << 20, p, 0, 1 << 20, None, None, 0, None), b"bad arguments")
        assert lib.trba_linear_int4_bytes(ins, outs, group, 0) == -1
    refused(lib.trba_linear_int4_create(4, 4, 32, None, None), b"bad arguments")
    for bad in ((None, 2, p, 0, 1), (p, 1, p, 0, 1), (p, 2, None, 0, 1), (p, 2, p, 1, 1), (p, 2, p, 0, 0)):
        refused(lib.trba_linear_int4_create_codes(4, 4, 32, *bad, None, None, 0, None), b"bad arguments")
    need = lib.trba_linear_int4_bytes(4, 4, 32, 0)
    assert need == 1024 + 4 * 16 * 4 + 16
    for at, size in ((64, need - 1), (72, need)):
        refused(lib.trba_linear_int4_create_codes(4, 4, 32, p, 2, p, 0, 1, None, C.c_void_p(at), size, None), b"storage")
    refused(lib.trba_linear_int4_forward(None, p, 0, 4, 1, p, 4, None, 0, None), b"bad arguments")
    assert lib.trba_linear_int4_workspace(None, 0, 9) == 0
    assert lib.trba_linear_int4_get(None, None, None, None) == -1 and lib.trba_linear_int4_param_count(None) == -1
    lib.trba_linear_int4_destroy(None)
    assert lib.trba_last_error() == 0


def test_python_refusals():
    w = np.zeros((4, 6), np.float32)
    for kw in (dict(group=16), dict(group=100), dict(in_features=0), dict(out_features=-1)):
        with pytest.raises(ValueError, match="LinearInt4"):
            LinearInt4(**{**dict(in_features=6, out_features=4, weight_f32=w), **kw})
    q, s = torch.zeros(4, 3, dtype=torch.uint8), torch.zeros(4, 1)
    for exc, word, args, kw in (
            (ValueError, "CUDA", (q, s), {}), (ValueError, "uint8", (q.int(), s), {}), (ValueError, "uint8", (q[:, :2], s), {}),
            (ValueError, "scales", (q, s.double()), {}), (ValueError, "scales", (q, s[:3]), {}), (ValueError, "scales", (q, s[:, :0]), {}),
            (ValueError, "bias", (q, s), dict(bias=torch.zeros(3))), (ValueError, "group", (q, s), dict(group=31)),
            (TypeError, "torch tensor", (q.numpy(), s), {})):
        with pytest.raises(exc, match=word):
            LinearInt4.from_codes(*args, **{**dict(in_features=6, group=32), **kw})


# ------------------------------------------------------------------- GPU --
def layer(outs, ins, group, scales, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (outs, -(-ins // 2)), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.rand(outs, -(-ins // group), generator=g, device="cuda").add_(0.05).mul_(0.1).to(DTYPES[scales])
    b = torch.randn(outs, generator=g, device="cuda") if bias else None
    return LinearInt4.from_codes(q, s, in_features=ins, group=group, bias=b), q, s, b


# |error|: products of a code and an activation are exact in f32; adding them
# up 16 at a time, ins / 16 additions and at most 20 more (scales, warps,
# bias), each off by at most 2^-23 of the sum of magnitudes (a tensor core
# truncates), and half a step of the output's type.
def check(y, x, q, s, b, ins, group):
    w = do.int4_weights(q.cpu().numpy(), s.float().cpu().numpy(), ins, group)
    xx = x.double().cpu().numpy().reshape(-1, ins)
    want, size = xx @ w.T, np.abs(xx) @ np.abs(w).T
    if b is not None:
        want, size = want + b.double().cpu().numpy(), size + np.abs(b.double().cpu().numpy())
    got = y.double().cpu().numpy().reshape(want.shape)
    tol = (ins / 16 + 20) * 2.0 ** -23 * size + torch.finfo(y.dtype).eps / 2 * np.abs(want)
    if y.dtype == torch.float16:
        tol += 2.0 ** -25  # half a step of its subnormals
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("outs,ins,group", [(1, 1, 32), (3, 2, 64), (7, 31, 32), (16, 33, 32), (17, 64, 64), (130, 256, 128),
                                            (64, 127, 64), (33, 129, 128), (100, 383, 384), (1000, 512, 64), (50, 1000, 256),
                                            (129, 4099, 32), (20, 16384, 128), (2600, 130, 128), (31, 2048, 2048)])
def test_forward_matches_oracle(outs, ins, group, dtype, lib, cuda):
    for k, rows in enumerate((1, 2, 3, 5, 8, 9, 17, 40, 64, 131)):
        lin, q, s, b = layer(outs, ins, group, ("f32", "f16")[k & 1], outs + rows, bias=k != 3)
        g = torch.Generator(device="cuda").manual_seed(rows)
        x = (torch.randn(rows, ins, generator=g, device="cuda") * torch.exp(torch.randn(ins, generator=g, device="cuda"))).to(DTYPES[dtype])
        y = lin.forward(x)
        assert y.shape == (rows, outs) and y.dtype == x.dtype
        check(y, x, q, s, b, ins, group)
        assert torch.equal(y, lin.forward(x))  # the same bits every time
        lin.close()
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_do_not_depend_on_each_other(dtype, cuda):
    """A row of infinities or NaN stays in its row; a zero row gives the bias."""
    outs, ins = 70, 300
    lin, q, s, b = layer(outs, ins, 64, "f32", 4)
    x = torch.randn(11, ins, device="cuda").to(DTYPES[dtype])
    x[2], x[5, 7], x[6, 9], x[9] = float("nan"), float("inf"), float("-inf"), 0.0
    y = lin.forward(x)
    ok = [0, 1, 3, 4, 7, 8, 10]
    check(y[ok], x[ok], q, s, b, ins, 64)
    assert torch.equal(y[9], b.to(y.dtype)) and y[2].isnan().all()
    for row, col, sign in ((5, 7, 1.0), (6, 9, -1.0)):
        code = ((q[:, col // 2] >> (4 * (col & 1))) & 15).int() - 8
        want = torch.where(code == 0, float("nan"), code.sign() * sign * float("inf"))
        assert torch.equal(y[row].float().nan_to_num(7.0, 1.0, -1.0), want.nan_to_num(7.0, 1.0, -1.0))


@pytest.mark.gpu
def test_extreme_f32_activations(cuda):
    """f32 activations keep all their bits: the largest, tiny ones, and ones that cancel."""
    outs, ins = 40, 256
    lin, q, s, _ = layer(outs, ins, 32, "f32", 6, bias=False)
    x = torch.zeros(5, ins, device="cuda")
    x[0, 3] = torch.finfo(torch.float32).max / 64
    x[1, 5] = 3.3e-30
    x[2] = 1.0 + torch.arange(ins, device="cuda") * 2.0 ** -23
    x[3] = torch.randn(ins, device="cuda")
    x[4] = 16777215.0
    check(lin.forward(x), x, q, s, None, ins, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("off,ldx,ldy", [(0, 200, 66), (1, 201, 67), (3, 208, 72), (8, 256, 128)])
def test_strides_and_leading_dimensions(off, ldx, ldy, dtype, cuda):
    t, rows, ins, outs = DTYPES[dtype], 13, 200, 66
    lin, q, s, b = layer(outs, ins, 64, "f16", off)
    buf = torch.full((rows * ldx + off + 8,), float("nan"), dtype=t, device="cuda")
    x = buf[off:off + rows * ldx].view(rows, ldx)[:, :ins]
    x.copy_(torch.randn(rows, ins, device="cuda"))
    ybuf = torch.full((rows * ldy + off + 8,), 9.0, dtype=t, device="cuda")
    y = ybuf[off:off + rows * ldy].view(rows, ldy)
    lin.forward(x, out=y[:, :outs])
    check(y[:, :outs], x, q, s, b, ins, 64)
    assert (y[:, outs:] == 9).all() and (ybuf[:off] == 9).all() and (ybuf[off + rows * ldy:] == 9).all()
    want = y[:, :outs].clone()
    assert torch.equal(lin.forward(x.contiguous()), want)
    assert torch.equal(lin.forward(x.contiguous().view(1, rows, ins))[0], want)
    assert torch.equal(lin.forward(x.T.contiguous().T), want)
    one = lin.forward(x[4])  # (the order of a row's sum may depend on the number of rows)
    assert one.shape == (outs,) and lin.forward(x[:0]).shape == (0, outs)
    check(one, x[4], q, s, b, ins, 64)


@pytest.mark.gpu
def test_quantised_layer(lib, cuda):
    rng = np.random.default_rng(5)
    for outs, ins, group in ((33, 300, 128), (130, 255, 64), (7, 1, 32), (64, 4096, 4096)):
        w = rng.standard_normal((outs, ins)).astype(np.float32)
        w[0, :32] = 0
        b = rng.standard_normal(outs).astype(np.float32)
        lin = LinearInt4(ins, outs, w, b, group=group)
        st = lin.state()
        q, s = do.int4_quantize(w, group)
        assert np.array_equal(st["scales"], s) and np.array_equal(st["codes"], q) and np.array_equal(st["bias"], b)
        assert lin.param_count() == outs * ins + outs
        x = torch.randn(4, ins, device="cuda")
        check(lin.forward(x), x, torch.from_numpy(q), torch.from_numpy(s), torch.from_numpy(b), ins, group)
    lin, q, s, b = layer(19, 77, 32, "f16", 1)
    st = lin.state()
    codes = q.cpu().numpy()
    codes[:, -1] = (codes[:, -1] & 15) | (st["codes"][:, -1] & 0xF0)  # behind the last input: no code
    assert np.array_equal(st["codes"], codes) and np.array_equal(st["scales"], s.float().cpu().numpy())
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
def test_layer_with_its_own_memory(lib, cuda):
    """create_codes without storage owns a copy: what it was made from may go."""
    lin, q, s, b = layer(37, 211, 64, "f16", 3)
    h = lib.trba_linear_int4_create_codes(211, 37, 64, C.c_void_p(q.data_ptr()), q.shape[1], C.c_void_p(s.data_ptr()), 2, s.shape[1],
                                          C.c_void_p(b.data_ptr()), None, 0, None)
    x = torch.randn(3, 211, device="cuda").bfloat16()
    want, y = lin.forward(x), torch.empty(3, 37, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    q.fill_(0), s.fill_(0)
    torch.cuda.synchronize()
    assert lib.trba_linear_int4_forward(h, C.c_void_p(x.data_ptr()), 1, 211, 3, C.c_void_p(y.data_ptr()), 37, None, 0, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(lin.forward(x), want)
    lib.trba_linear_int4_destroy(h)


@pytest.mark.gpu
def test_layer_dropped_while_another_stream_reads_it(cuda):
    """The memory of a layer made on one stream is not handed out again before
    a call on another is done with it."""
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    kept, q, s, b = layer(2000, 4096, 128, "f16", 5)
    x = torch.randn(24, 4096, device="cuda").half()
    want = kept.forward(x)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(made):
            lin = LinearInt4.from_codes(q, s, in_features=4096, group=128, bias=b)
            size = lin.storage.numel()
        used.wait_stream(made)
        ys = [lin.forward(x, stream=used) for _ in range(20)]
        del lin
        with torch.cuda.stream(made):
            junk = torch.empty(size, dtype=torch.uint8, device="cuda").fill_(0x77)
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in ys)
        del junk


@pytest.mark.gpu
def test_forward_refusals(lib, cuda):
    lin, *_ = layer(8, 40, 32, "f32", 0)
    x = torch.zeros(2, 40, device="cuda")
    for exc, word, args, kw in ((TypeError, "float32", (x.double(),), {}), (ValueError, "in_features", (x[:, :39],), {}),
                                (ValueError, "CUDA", (x.cpu(),), {}), (ValueError, "out must be", (x,), dict(out=x)),
                                (ValueError, "apart", (x,), dict(out=torch.zeros(1, 8, device="cuda").expand(2, 8))),
                                (TypeError, "torch tensor", (x.cpu().numpy(),), {}),
                                (ValueError, "overlaps", (x,), dict(out=x.view(-1)[30:46].view(2, 8)))):
        with pytest.raises(exc, match=word):
            lin.forward(*args, **kw)
    lib.trba_clear_error()
    p = C.c_void_p(x.data_ptr())
    for args, word in (((None, 0, 40, 1, p, 8), b"bad arguments"), ((p, 0, 39, 1, p, 8), b"bad arguments"), ((p, 0, 40, -1, p, 8), b"bad arguments"),
                       ((p, 0, 40, 1, p, 7), b"bad arguments"), ((p, 3, 40, 1, p, 8), b"element type"),
                       ((C.c_void_p(x.data_ptr() + 2), 0, 40, 1, p, 8), b"not aligned"), ((p, 0, 40, 9, p, 8), b"workspace")):
        assert lib.trba_linear_int4_forward(lin.h, *args, None, 0, None) == -1 and word in lib.trba_last_error_string()
        lib.trba_clear_error()
    assert lib.trba_linear_int4_forward(lin.h, None, 0, 40, 0, None, 8, None, 0, None) == 0
    assert lib.trba_linear_int4_workspace(lin.h, 0, 1) == 0 < lib.trba_linear_int4_workspace(lin.h, 0, 9)
    lin.close()
    lin.close()


@pytest.mark.gpu
def test_captured_on_two_streams(cuda):
    """Two graphs of one layer run at once and on new inputs."""
    lin, q, s, b = layer(300, 1111, 64, "f16", 8)
    xs = [torch.randn(5, 1111, device="cuda").bfloat16() for _ in range(4)]
    want = [lin.forward(x) for x in xs]
    graphs = []
    for k in range(2):
        buf = xs[k].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = lin.forward(buf)
        graphs.append((g, buf, y, torch.cuda.Stream()))
    for r in range(2):
        for k, (g, buf, y, st) in enumerate(graphs):
            with torch.cuda.stream(st):
                buf.copy_(xs[2 * r + k])
                g.replay()
        torch.cuda.synchronize()
        for k, (_, _, y, _) in enumerate(graphs):
            assert torch.equal(y, want[2 * r + k])
    st = torch.cuda.Stream()
    y = lin.forward(xs[0], stream=st)
    st.synchronize()
    assert torch.equal(y, want[0])


@pytest.mark.gpu
def test_beam_search_through_the_layer(lib, cuda):
    """The operators as they are used together: an LSTM decoder whose gates and
    vocabulary are 4-bit layers, searched with beams; every step's logits
    against f64, every choice against the oracle on those logits."""
    from test_decode import check_step
    L, K, V, H, T, eos = 3, 4, 131, 96, 9, 2
    rng = np.random.default_rng(12)
    wg, wo = rng.standard_normal((4 * H, 2 * H)).astype(np.float32) * 0.2, rng.standard_normal((V, H)).astype(np.float32)
    gates = LinearInt4(2 * H, 4 * H, wg, rng.standard_normal(4 * H).astype(np.float32), group=64)
    gen = LinearInt4(H, V, wo, None, group=32)
    emb = torch.randn(V, H, device="cuda")
    wo_q = do.int4_quantize(wo, 32)
    h = torch.zeros(L * K, H, device="cuda")
    c = torch.zeros_like(h)
    scores = torch.full((L, K), float("-inf"), device="cuda")
    scores[:, 0] = 0
    fin, tokens = torch.zeros(L, K, dtype=torch.bool, device="cuda"), torch.ones(L, K, dtype=torch.int32, device="cuda")
    hist = []
    for _ in range(T):
        i, f, g, o = gates.forward(torch.cat([emb[tokens.view(-1).long()], h], 1)).chunk(4, 1)
        c = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(g)
        h = torch.sigmoid(o) * torch.tanh(c)
        logits = gen.forward(h)
        check(logits, h, torch.from_numpy(wo_q[0]), torch.from_numpy(wo_q[1]), None, H, 32)
        step = decode.beam_select(logits, scores, fin, eos=eos)
        check_step(step, logits, scores, fin, eos)
        before = h
        h, c = decode.beam_reorder([h, c], step.parents)
        assert torch.equal(h.view(L, K, H)[1, 2], before.view(L, K, H)[1, step.parents[1, 2]])
        scores, tokens, fin = step.scores, step.tokens, step.finished
        hist.append(step)
    seq, n = decode.beam_sequences(torch.stack([s.tokens for s in hist]), torch.stack([s.parents for s in hist]), eos=eos)
    want = do.beam_sequences(*(np.stack([x.cpu().numpy() for x in xs]) for xs in
                               ([s.tokens for s in hist], [s.parents for s in hist])), eos, 0)
    assert np.array_equal(seq.cpu().numpy(), want[0]) and np.array_equal(n.cpu().numpy(), want[1])
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_output_beside_its_input(dtype, cuda):
    """x and y as columns of one buffer, as layers that append to their input keep them."""
    for rows, ins, outs in ((1, 40, 24), (5, 203, 70), (20, 203, 70)):
        lin, q, s, b = layer(outs, ins, 32, "f32", rows)
        buf = torch.randn(rows, ins + outs + 3, device="cuda").to(DTYPES[dtype])
        x, rest = buf[:, :ins].clone(), buf[:, ins + outs:].clone()
        lin.forward(buf[:, :ins], out=buf[:, ins:ins + outs])
        check(buf[:, ins:ins + outs], x, q, s, b, ins, 32)
        assert torch.equal(buf[:, :ins], x) and torch.equal(buf[:, ins + outs:], rest)
        with pytest.raises(ValueError, match="overlaps"):
            lin.forward(buf[:, :ins], out=buf[:, ins - 1:ins - 1 + outs])


@pytest.mark.gpu
def test_negated_views(cuda):
    """torch's lazily negated views are read as the values they stand for."""
    lin, q, s, b = layer(30, 100, 32, "f32", 2)
    x = torch.randn(4, 100, device="cuda")
    want = lin.forward(x)
    assert torch.equal(lin.forward(torch._neg_view(-x)), want)
    other = LinearInt4.from_codes(q, torch._neg_view(-s), in_features=100, group=32, bias=torch._neg_view(-b))
    assert torch.equal(other.forward(x), want)
    with pytest.raises(ValueError, match="out must be"):
        lin.forward(x, out=torch._neg_view(torch.zeros(4, 30, device="cuda")))


# ------------------------------------------------- GPU: what large sizes do --
def check_rows(y, x, q, s, ins, group, at):
    """check() for the outputs `at` alone."""
    check(y[:, at].contiguous(), x, q[at], s[at], None, ins, group)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("outs,ins,group", [(50001, 300, 32), (40000, 643, 128)])
def test_many_tiles_a_block(outs, ins, group, dtype, lib, cuda):
    """More than eight columns through more tiles than the device has blocks for
    at once: stages and partial sums go on from one group of tiles to the next."""
    for rows in (9, 17, 24, 40, 61):
        lin, q, s, b = layer(outs, ins, group, ("f32", "f16")[rows & 1], rows)
        g = torch.Generator(device="cuda").manual_seed(rows)
        x = torch.randn(rows, ins, generator=g, device="cuda").to(DTYPES[dtype])
        check(lin.forward(x), x, q, s, b, ins, group)
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows", [("f16", 8), ("bf16", 7), ("f32", 2)])
@pytest.mark.parametrize("outs,ins,group", [(5000, 16384, 128), (40001, 16001, 32)])
def test_tiles_and_slabs(outs, ins, group, dtype, rows, lib, cuda):
    """Few columns, several tiles a block, and more inputs than are staged at
    once: sums of all its tiles wait between the slabs."""
    lin, q, s, _ = layer(outs, ins, group, "f16", rows, bias=False)
    x = torch.randn(rows, ins, generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda").to(DTYPES[dtype])
    y = lin.forward(x)
    at = torch.cat([torch.arange(0, outs, 37), torch.arange(40), torch.arange(outs - 40, outs)]).cuda()
    check_rows(y, x, q, s, ins, group, at)
    assert torch.equal(y, lin.forward(x))
    # every output: by the same layer in parts that have a tile or two a block
    for n0 in range(0, outs, 4096):
        n1 = min(outs, n0 + 4096)
        part = LinearInt4.from_codes(q[n0:n1], s[n0:n1], in_features=ins, group=group)
        size = (x.double().abs() @ torch.full((ins, 1), 8 * float(s.max()), dtype=torch.float64, device="cuda")).max()
        tol = 2 * ((ins / 16 + 20) * 2.0 ** -23 * size + torch.finfo(x.dtype).eps / 2 * y.double().abs().max())
        assert (part.forward(x).double() - y[:, n0:n1].double()).abs().max() <= tol
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
def test_more_blocks_than_processors(lib, cuda):
    """So many outputs that their sums leave no room for a slab: the grid grows."""
    outs, ins, group, rows = 600007, 8500, 128, 8
    lin, q, s, _ = layer(outs, ins, group, "f16", 3, bias=False)
    x = torch.randn(rows, ins, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    y = lin.forward(x)
    at = torch.cat([torch.arange(0, outs, 997), torch.arange(outs - 20, outs)]).cuda()
    check_rows(y, x, q, s, ins, group, at)
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
def test_codes_and_scales_with_wider_rows(lib, cuda):
    """create_codes with row strides above the rows' sizes, at an odd address of the codes."""
    outs, ins, group = 45, 211, 64
    wide = torch.randint(0, 256, (outs * 130 + 7,), dtype=torch.uint8, device="cuda")
    for dtype, off, ld, lds in ((torch.float32, 0, 106, 4), (torch.float16, 3, 113, 7), (torch.float16, 4, 128, 5), (torch.float32, 1, 130, 9)):
        q = wide[off:off + outs * ld].view(outs, ld)[:, :106]
        s = (torch.rand(outs, lds, device="cuda") * 0.1 + 0.01).to(dtype)
        h = lib.trba_linear_int4_create_codes(ins, outs, group, C.c_void_p(q.data_ptr()), ld, C.c_void_p(s.data_ptr()),
                                              0 if dtype == torch.float32 else 2, lds, None, None, 0, None)
        lin = LinearInt4.from_codes(q.contiguous(), s[:, :4].contiguous(), in_features=ins, group=group)
        x = torch.randn(3, ins, device="cuda").bfloat16()
        want, y = lin.forward(x), torch.empty(3, outs, dtype=torch.bfloat16, device="cuda")
        assert lib.trba_linear_int4_forward(h, C.c_void_p(x.data_ptr()), 1, ins, 3, C.c_void_p(y.data_ptr()), outs, None, 0, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        check(y, x, q, s[:, :4], None, ins, group)
        lib.trba_linear_int4_destroy(h)
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
def test_memory_of_a_dropped_layer_waits_for_the_reading_stream(cuda):
    """While calls on another stream are pending, the memory of the layer that
    they read is not handed out again on the stream that made it."""
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    kept, q, s, b = layer(2000, 4096, 128, "f16", 5)
    x = torch.randn(24, 4096, device="cuda").half()
    want = kept.forward(x)
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for read in (False, True):
        with torch.cuda.stream(made):
            lin = LinearInt4.from_codes(q, s, in_features=4096, group=128, bias=b)
        size, ptr = lin.storage.numel(), lin.storage.data_ptr()
        used.wait_stream(made)
        with torch.cuda.stream(used):
            for _ in range(40):  # tens of ms ahead of the layer's calls
                busy = torch.tanh(busy @ busy)
        ys = [lin.forward(x, stream=used) for _ in range(20)] if read else []
        done = torch.cuda.Event()
        done.record(used)
        del lin
        with torch.cuda.stream(made):
            again = [torch.empty(size, dtype=torch.uint8, device="cuda").fill_(0x77) for _ in range(3)]
        assert not done.query()
        # (without a reader the block comes back at once: the check below can fail)
        assert (ptr in [t.data_ptr() for t in again]) == (not read)
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in ys)
        del again


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 9])
def test_tiny_activations(rows, cuda):
    """Subnormal activations count in all types; of an f32 activation only what
    lies below 2^-133 (the last place of a bf16) is dropped."""
    outs, ins = 24, 256
    lin, q, s, _ = layer(outs, ins, 32, "f32", 9, bias=False)
    k = torch.randint(-500, 500, (rows, ins), generator=torch.Generator().manual_seed(rows)).cuda()
    w = do.int4_weights(q.cpu().numpy(), s.cpu().numpy(), ins, 32)
    for dtype, unit, dropped in ((torch.float16, 2.0 ** -24, 0.0), (torch.bfloat16, 2.0 ** -133, 0.0), (torch.float32, 2.0 ** -133, 0.0),
                                 (torch.float32, 2.0 ** -143, 2.0 ** -133), (torch.float32, 2.0 ** -149, 2.0 ** -133)):
        x = (k.double() * unit).to(dtype)
        xx = x.double().cpu().numpy()
        want, size = xx @ w.T, np.abs(xx) @ np.abs(w).T
        # check()'s rule, what is dropped times its weight, and half a step of the
        # output's and the sums' subnormals (ins / 16 + 20 additions, 2^-150 each)
        lost = dropped * np.abs(w).sum(1) + (ins / 16 + 20) * 2.0 ** -149 + {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}.get(dtype, 2.0 ** -150)
        tol = (ins / 16 + 20) * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * np.abs(want) + lost
        err = np.abs(lin.forward(x).double().cpu().numpy() - want)
        assert (err <= tol).all(), (dtype, unit, (err / tol).max())
        if dtype != torch.float16 and unit == 2.0 ** -133:
            assert np.abs(want).max() > 100 * np.max(lost)  # (values that would show if they were taken as zero)


@pytest.mark.gpu
@pytest.mark.parametrize("ins", [1 << 30, (1 << 30) - 129])
def test_most_inputs(ins, lib, cuda):
    """The most inputs that a layer takes: the staged activations of a row are
    counted in 64 bits.  Three inputs count, the rest are zero."""
    outs, rows = 3, 2
    q = torch.full((outs, -(-ins // 2)), 0x88, dtype=torch.uint8, device="cuda")
    s = torch.ones(outs, 1, device="cuda")
    at = [0, ins // 2 + 77, ins - 1]
    code = torch.randint(0, 16, (outs, 3), generator=torch.Generator().manual_seed(1), dtype=torch.uint8).cuda()
    for j, k in enumerate(at):
        q[:, k // 2] = (0x80 | code[:, j]) if k % 2 == 0 else (8 | code[:, j] << 4)
    lin = LinearInt4.from_codes(q, s, in_features=ins, group=1 << 30)
    del q
    x = torch.zeros(rows, ins, dtype=torch.bfloat16, device="cuda")
    x[:, at] = torch.tensor([[1.0, 2.0, -3.0], [0.5, -4.0, 8.0]], device="cuda").bfloat16()
    want = x[:, at].float() @ (code.float() - 8).T
    assert torch.equal(lin.forward(x).float(), want.bfloat16().float())
    assert torch.equal(lin.forward(x[:1]).float(), want[:1].bfloat16().float())
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_most_rows(dtype, lib, cuda):
    outs, ins, rows = 40, 64, 1000000
    lin, q, s, b = layer(outs, ins, 32, "f32", 1)
    x = torch.randn(rows, ins, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(DTYPES[dtype])
    y = lin.forward(x)
    w = torch.from_numpy(do.int4_weights(q.cpu().numpy(), s.cpu().numpy(), ins, 32)).cuda()
    want, size = x.double() @ w.T + b, x.double().abs() @ w.abs().T + b.abs()
    tol = (ins / 16 + 20) * 2.0 ** -23 * size + torch.finfo(y.dtype).eps / 2 * want.abs() + 2.0 ** -25  # as in check()
    assert ((y.double() - want).abs() <= tol).all()
    with pytest.raises(ValueError, match="million"):
        lin.forward(x[:1].expand(rows + 1, ins))
    assert lib.trba_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,outs,ins", [("f16", 40, 1000, 4000), ("bf16", 16, 3000, 1111), ("f32", 9, 130, 2048)])
def test_many_columns_captured_on_two_streams(dtype, rows, outs, ins, cuda):
    """As test_captured_on_two_streams, for the two launches of many columns
    (inputs split over clusters in the first and the last)."""
    lin, q, s, b = layer(outs, ins, 64, "f16", 8)
    xs = [torch.randn(rows, ins, device="cuda").to(DTYPES[dtype]) for _ in range(4)]
    want = [lin.forward(x) for x in xs]
    graphs = []
    for k in range(2):
        buf = xs[k].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ys = [lin.forward(buf) for _ in range(4)]
        graphs.append((g, buf, ys, torch.cuda.Stream()))
    for r in range(2):
        for k, (g, buf, _, st) in enumerate(graphs):
            with torch.cuda.stream(st):
                buf.copy_(xs[2 * r + k])
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for k, (_, _, ys, _) in enumerate(graphs):
            assert all(torch.equal(y, want[2 * r + k]) for y in ys)
