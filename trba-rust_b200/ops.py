"""Python mirror of the reference's INT8 operator API over libtrba_b200
(include/trba_ops.h): LinearInt8 (src/linear.rs), LSTMInt8 and BiLSTMInt8
(src/bilstm.rs).  Method names, argument meaning and return values follow
the Rust structs; weights are injected (the reference draws them from
rand::thread_rng), and all state lives on the device.

    lin = LinearInt8(in_features, out_features, weight_f32, bias)
    out = lin.forward(inp_int8)                   # [rows*out] int32
    clip = lin.backward(inp_f32, grad_out, lr, mom)

LinearInt4, beside them, is a linear layer with 4-bit weights for decoding; it
works on torch CUDA tensors.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from .ffi import lib


def _p(a: np.ndarray):
    assert a.flags.c_contiguous
    return C.c_void_p(a.ctypes.data)


def _err(L, what):
    return RuntimeError(f"{what}: " + L.trba_last_error_string().decode())


class LinearInt8:
    """src/linear.rs:12-180."""

    def __init__(self, in_features: int, out_features: int, weight_f32: np.ndarray, bias: np.ndarray | None = None):
        self.L = lib()
        self.in_features, self.out_features = in_features, out_features
        w = np.ascontiguousarray(weight_f32, np.float32).reshape(out_features * in_features)
        b = None if bias is None else np.ascontiguousarray(bias, np.float32).reshape(out_features)
        self.h = self.L.trba_linear_int8_create(in_features, out_features, _p(w), None if b is None else _p(b))
        if not self.h:
            raise _err(self.L, "LinearInt8::new")

    def close(self):
        if getattr(self, "h", None):
            self.L.trba_linear_int8_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _state(self):
        n = self.in_features * self.out_features
        w, q = np.empty(n, np.float32), np.empty(n, np.int8)
        b, g = np.empty(self.out_features, np.float32), np.empty(n, np.float32)
        if self.L.trba_linear_int8_get(self.h, _p(w), _p(q), _p(b), _p(g)) != 0:
            raise _err(self.L, "LinearInt8 state")
        return w, q, b, g

    @property
    def weight_f32(self) -> np.ndarray:
        return self._state()[0]

    @weight_f32.setter
    def weight_f32(self, w):
        w = np.ascontiguousarray(w, np.float32).reshape(-1)
        if self.L.trba_linear_int8_set(self.h, _p(w), None) != 0:
            raise _err(self.L, "LinearInt8 set weights")

    @property
    def weight_int8(self) -> np.ndarray:
        return self._state()[1]

    @property
    def bias(self) -> np.ndarray:
        return self._state()[2]

    @property
    def grad_f32(self) -> np.ndarray:
        return self._state()[3]

    def requantize(self):
        self.L.trba_linear_int8_requantize(self.h, None)

    def forward(self, inp: np.ndarray) -> np.ndarray:
        """[rows, in] int8 -> [rows*out] int32 (src/linear.rs:66-115)."""
        inp = np.ascontiguousarray(inp, np.int8).reshape(-1)
        if inp.size == 0 or inp.size % self.in_features:
            raise ValueError(f"LinearInt8::forward: input {inp.size} is not a multiple of in_features "
                             f"{self.in_features}")
        out = np.empty(inp.size // self.in_features * self.out_features, np.int32)
        if self.L.trba_linear_int8_forward_host(self.h, _p(inp), inp.size, _p(out)) != 0:
            raise _err(self.L, "LinearInt8::forward")
        return out

    def backward(self, inp: np.ndarray, grad_out: np.ndarray, lr: float, mom: float) -> float:
        """FP32 backward + SGD with global-norm clipping; returns the clip
        factor (src/linear.rs:121-175)."""
        inp = np.ascontiguousarray(inp, np.float32).reshape(-1)
        go = np.ascontiguousarray(grad_out, np.float32).reshape(-1)
        return float(self.L.trba_linear_int8_backward_host(self.h, _p(inp), inp.size, _p(go), go.size,
                                                           float(lr), float(mom)))

    def param_count(self) -> int:
        return int(self.L.trba_linear_int8_param_count(self.h))


class LinearInt4:
    """Linear layer with 4-bit weights and one scale per `group` inputs, for
    the few rows of a decoding step (include/trba_ops.h):

        lin = LinearInt4(in_features, out_features, weight_f32, bias, group=128)
        y = lin.forward(x)     # torch CUDA tensors, [rows, in] -> [rows, out]

    An operator for serving: forward records no graph, and y requires no
    gradient although x may.  No counterpart in the reference."""

    def __init__(self, in_features: int, out_features: int, weight_f32: np.ndarray, bias: np.ndarray | None = None,
                 group: int = 128):
        """Quantises f32 weights [out, in] (host): per group, scale = max |w| /
        7 and code - 8 = round(w / scale)."""
        self._check_sizes(in_features, out_features, group)
        w = np.ascontiguousarray(weight_f32, np.float32).reshape(out_features * in_features)
        b = None if bias is None else np.ascontiguousarray(bias, np.float32).reshape(out_features)
        self._own(in_features, out_features, group,
                  lib().trba_linear_int4_create(in_features, out_features, group, _p(w), None if b is None else _p(b)))

    @staticmethod
    def _check_sizes(in_features, out_features, group):
        if not (1 <= in_features <= 1 << 30 and 1 <= out_features <= 1 << 30):
            raise ValueError(f"LinearInt4: sizes must be 1 to 2**30, got {in_features} -> {out_features}")
        if group not in (32, 64) and (group < 128 or group % 128):
            raise ValueError(f"LinearInt4: group must be 32, 64 or a multiple of 128, got {group}")

    def _own(self, in_features, out_features, group, handle):
        import torch
        from . import decode
        self.L, self.torch, self.decode = lib(), torch, decode
        self.in_features, self.out_features, self.group, self.h = in_features, out_features, group, handle
        if not handle:
            raise _err(self.L, "LinearInt4")
        self.device = torch.device("cuda", torch.cuda.current_device())

    @classmethod
    def from_codes(cls, codes, scales, *, in_features: int, group: int = 128, bias=None) -> "LinearInt4":
        """From quantised weights on the GPU: codes [out, ceil(in / 2)] uint8,
        the even input's code in the low half; scales [out, ceil(in / group)]
        float32 or float16; bias [out] float32 or None.  W = (code - 8) *
        scale.  The tensors are copied, in the order of torch's current stream;
        a layer used on another stream is made there or waited for first."""
        import torch
        from .decode import DTYPE_CODES, _check_cuda, _check_tensors, _on, _plain, _raw_stream
        _check_tensors(codes=codes, scales=scales, bias=bias)
        if in_features < 1 or codes.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[1] != -(-in_features // 2):
            raise ValueError(f"codes must be a uint8 tensor [out, {-(-in_features // 2)}]")
        out_features = codes.shape[0]
        cls._check_sizes(in_features, out_features, group)
        if scales.dtype not in (torch.float32, torch.float16) or tuple(scales.shape) != (out_features,
                                                                                       -(-in_features // group)):
            raise ValueError(f"scales must be float32 or float16 [{out_features}, {-(-in_features // group)}]")
        if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (out_features,)):
            raise ValueError(f"bias must be float32 [{out_features}]")
        device = codes.device
        for name, t in (("codes", codes), ("scales", scales), ("bias", bias)):
            if t is not None:
                _check_cuda(name, t, device)
        self = cls.__new__(cls)
        with _on(device, None):
            codes, scales = _plain(codes).contiguous(), _plain(scales).contiguous()
            bias = None if bias is None else _plain(bias).contiguous()
            need = lib().trba_linear_int4_bytes(in_features, out_features, group, DTYPE_CODES[scales.dtype])
            storage = torch.empty(need, dtype=torch.uint8, device=device)
            self.home = _raw_stream(device.index)  # the stream the storage belongs to
            self._own(in_features, out_features, group, lib().trba_linear_int4_create_codes(
                in_features, out_features, group, codes.data_ptr(), codes.shape[1], scales.data_ptr(),
                DTYPE_CODES[scales.dtype], scales.shape[1], None if bias is None else bias.data_ptr(),
                storage.data_ptr(), need, self.home))
            self.storage = storage
        return self

    storage = None  # torch's memory of a layer made by from_codes

    def close(self):
        if getattr(self, "h", None):
            self.L.trba_linear_int4_destroy(self.h)
            self.h = self.storage = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, x, out=None, stream=None):
        """[rows, in] -> [rows, out] of the same type (float32, bfloat16 or
        float16); leading dimensions of x are rows.  Runs on torch's current
        stream, or on `stream` (a torch.cuda.Stream).  `out` must share no
        memory with x."""
        torch, decode = self.torch, self.decode
        if not self.h:
            raise RuntimeError("LinearInt4::forward: the layer is closed")
        if not isinstance(x, torch.Tensor) or out is not None:
            decode._check_tensors(x=x, out=out)
        code = decode.DTYPE_CODES.get(x.dtype)
        if code is None:
            raise TypeError(f"LinearInt4::forward: x must be float32, bfloat16 or float16, got {x.dtype}")
        ins, outs, device = self.in_features, self.out_features, self.device
        if x.dim() < 1 or x.shape[-1] != ins:
            raise ValueError(f"LinearInt4::forward: x {tuple(x.shape)} does not end in in_features {ins}")
        shape = x.shape[:-1] + (outs,)
        if x.device != device:
            decode._check_cuda("x", x, device)
        if stream is not None or device.index != decode._current_device():
            with decode._on(device, stream):
                return self.forward(x, out)
        if x.is_neg():
            x = decode._plain(x)
        if x.dim() != 2:
            x = x.reshape(-1, ins)
        rows = x.shape[0]
        if not x.is_contiguous() and ((ins > 1 and x.stride(1) != 1) or (rows > 1 and x.stride(0) < ins)):
            x = x.contiguous()
        if out is None:
            out = torch.empty(shape, dtype=x.dtype, device=device)
            ldy = outs
        else:
            decode._check_cuda("out", out, device)
            if out.shape != shape or out.dtype != x.dtype or out.is_neg():
                raise ValueError(f"LinearInt4::forward: out must be {x.dtype} {tuple(shape)}")
            if out.dim() != 2 and not out.is_contiguous():
                raise ValueError("LinearInt4::forward: out must be contiguous")
            ldy = out.stride(0) if out.dim() == 2 and rows > 1 else outs
            if ldy < outs or (outs > 1 and out.stride(-1) != 1):
                raise ValueError("LinearInt4::forward: the rows of out must be contiguous and apart")
            decode._check_apart({"LinearInt4::forward: out": out}, {"x": x})
        if rows > 1000000:
            raise ValueError("LinearInt4::forward: at most a million rows")
        if rows:
            raw = decode._raw_stream(device.index)
            if self.storage is not None and raw != self.home:
                self.storage.record_stream(torch.cuda.current_stream(device))  # not to be reused before this call is done
            need = self.L.trba_linear_int4_workspace(self.h, code, rows) if rows > 2 else 0
            work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            rc = self.L.trba_linear_int4_forward(self.h, x.data_ptr(), code, x.stride(0) if rows > 1 else ins, rows,
                                                 out.data_ptr(), ldy, work.data_ptr() if need else None, need, raw)
            if rc:
                raise _err(self.L, "LinearInt4::forward")
        return out

    def state(self) -> dict:
        """Host copies: codes [out, ceil(in / 2)] uint8, scales [out, groups]
        float32, bias [out] float32."""
        if not self.h:
            raise RuntimeError("LinearInt4 state: the layer is closed")
        n, g = self.out_features, -(-self.in_features // self.group)
        q, s = np.empty((n, -(-self.in_features // 2)), np.uint8), np.empty((n, g), np.float32)
        b = np.empty(n, np.float32)
        with self.torch.cuda.device(self.device):
            rc = self.L.trba_linear_int4_get(self.h, _p(q), _p(s), _p(b))
        if rc != 0:
            raise _err(self.L, "LinearInt4 state")
        return {"codes": q, "scales": s, "bias": b}

    def param_count(self) -> int:
        return int(self.L.trba_linear_int4_param_count(self.h))


class LSTMInt8:
    """src/bilstm.rs:13-178.  forward_step etc. take host numpy arrays."""

    def __init__(self, input_size: int, hidden_size: int, w_ih: np.ndarray, w_hh: np.ndarray,
                 bias: np.ndarray | None = None):
        self.L = lib()
        self.input_size, self.hidden_size = input_size, hidden_size
        wi = np.ascontiguousarray(w_ih, np.float32).reshape(-1)
        wh = np.ascontiguousarray(w_hh, np.float32).reshape(-1)
        b = None if bias is None else np.ascontiguousarray(bias, np.float32).reshape(-1)
        self.h = self.L.trba_lstm_int8_create(input_size, hidden_size, _p(wi), _p(wh), None if b is None else _p(b))
        if not self.h:
            raise _err(self.L, "LSTMInt8::new")

    def close(self):
        if getattr(self, "h", None):
            self.L.trba_lstm_int8_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def state(self):
        G, I, H = 4 * self.hidden_size, self.input_size, self.hidden_size
        wi, qi = np.empty(G * I, np.float32), np.empty(G * I, np.int8)
        wh, qh = np.empty(G * H, np.float32), np.empty(G * H, np.int8)
        b = np.empty(G, np.float32)
        if self.L.trba_lstm_int8_get(self.h, _p(wi), _p(qi), _p(wh), _p(qh), _p(b)) != 0:
            raise _err(self.L, "LSTMInt8 state")
        return {"weight_ih_f32": wi, "weight_ih_int8": qi, "weight_hh_f32": wh, "weight_hh_int8": qh, "bias": b}

    def requantize(self):
        self.L.trba_lstm_int8_requantize(self.h, None)

    def forward_step(self, x_int8, h_prev, c_prev, batch_size: int):
        """src/bilstm.rs:72-117 -> (h_new, c_new) as float32 [batch*hidden]."""
        import torch
        x = torch.from_numpy(np.ascontiguousarray(x_int8, np.int8).reshape(-1)).cuda()
        hp = torch.from_numpy(np.ascontiguousarray(h_prev, np.float32).reshape(-1)).cuda()
        cp = torch.from_numpy(np.ascontiguousarray(c_prev, np.float32).reshape(-1)).cuda()
        hn = torch.empty(batch_size * self.hidden_size, dtype=torch.float32, device="cuda")
        cn = torch.empty_like(hn)
        rc = self.L.trba_lstm_int8_forward_step(self.h, C.c_void_p(x.data_ptr()), C.c_void_p(hp.data_ptr()),
                                                C.c_void_p(cp.data_ptr()), batch_size, C.c_void_p(hn.data_ptr()),
                                                C.c_void_p(cn.data_ptr()), None)
        if rc != 0:
            raise _err(self.L, "LSTMInt8::forward_step")
        return hn.cpu().numpy(), cn.cpu().numpy()

    def _proj(self, fn, a, batch, k):
        import torch
        t = torch.from_numpy(np.ascontiguousarray(a, np.int8).reshape(-1)).cuda()
        out = torch.empty(batch * 4 * self.hidden_size, dtype=torch.int32, device="cuda")
        if fn(self.h, C.c_void_p(t.data_ptr()), batch, C.c_void_p(out.data_ptr()), None) != 0:
            raise _err(self.L, "LSTMInt8 projection")
        return out.cpu().numpy()

    def i2h_forward(self, x_int8, batch: int):
        return self._proj(self.L.trba_lstm_int8_i2h_forward, x_int8, batch, self.input_size)

    def h2h_forward(self, h_int8, batch: int):
        return self._proj(self.L.trba_lstm_int8_h2h_forward, h_int8, batch, self.hidden_size)

    @staticmethod
    def gemm_int8(a, b, m: int, n: int, k: int) -> np.ndarray:
        """src/bilstm.rs:132-173 on compact operands."""
        import torch
        L = lib()
        ta = torch.from_numpy(np.ascontiguousarray(a, np.int8).reshape(-1)).cuda()
        tb = torch.from_numpy(np.ascontiguousarray(b, np.int8).reshape(-1)).cuda()
        out = torch.empty(m * n, dtype=torch.int32, device="cuda")
        if L.trba_gemm_int8_compact(C.c_void_p(ta.data_ptr()), C.c_void_p(tb.data_ptr()),
                                    C.c_void_p(out.data_ptr()), m, n, k, None) != 0:
            raise _err(L, "LSTMInt8::gemm_int8")
        return out.cpu().numpy()

    def param_count(self) -> int:
        return int(self.L.trba_lstm_int8_param_count(self.h))


class BiLSTMInt8:
    """src/bilstm.rs:180-256."""

    def __init__(self, forward: LSTMInt8, backward: LSTMInt8):
        self.forward_lstm, self.backward_lstm = forward, backward
        self.hidden_size = forward.hidden_size

    def forward(self, x_seq_int8, batch_size: int, seq_len: int) -> np.ndarray:
        """x [seq_len, batch, input] int8 -> [batch * 2*hidden] float32."""
        import torch
        L = lib()
        need = seq_len * batch_size * self.forward_lstm.input_size
        x = np.ascontiguousarray(x_seq_int8, np.int8).reshape(-1)
        if x.size < need:
            raise ValueError(f"BiLSTM::forward: input is {x.size} bytes, need {need}")
        t = torch.from_numpy(x[:max(need, 1)].copy()).cuda()
        out = torch.empty(batch_size * 2 * self.hidden_size, dtype=torch.float32, device="cuda")
        if L.trba_bilstm_int8_forward(self.forward_lstm.h, self.backward_lstm.h, C.c_void_p(t.data_ptr()),
                                      batch_size, seq_len, C.c_void_p(out.data_ptr()), None) != 0:
            raise _err(L, "BiLSTMInt8::forward")
        return out.cpu().numpy()

    def param_count(self) -> int:
        return self.forward_lstm.param_count() + self.backward_lstm.param_count()
