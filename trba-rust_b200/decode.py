"""Beam-search operators on torch CUDA tensors (include/trba_decode.h).

    step = beam_select(logits, scores, finished, eos=2)   # scores, tokens, parents, finished
    h, c = beam_reorder([h, c], step.parents)             # the states follow their beams
    seqs, lengths = beam_sequences(tokens, parents, eos=2)

Work is queued on torch's current stream of the tensors' device, or on
``stream`` (a torch.cuda.Stream); outputs and workspaces belong to that
stream.  As with torch's own operators, inputs that another stream writes have
to be waited for, and kept, by the caller.  Arguments are checked here: a
ValueError or TypeError means that nothing ran.  These are operators for
serving: they record no graph, and what they return for inputs that require
gradients requires none.
"""
from __future__ import annotations

import functools
import math
import struct
from typing import NamedTuple, Sequence

import torch

from .ffi import lib

MAX_BEAMS = 32
MOST_PARTS = 2 ** 31 - 1 - 2 ** 20  # contiguous parts of a state's rows (of at most 1024 bytes each)
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class BeamStep(NamedTuple):
    scores: torch.Tensor    # [lines, beams] float32
    tokens: torch.Tensor    # [lines, beams] int32
    parents: torch.Tensor   # [lines, beams] int32
    finished: torch.Tensor  # [lines, beams] bool


def _fail(L, what, rc):
    raise RuntimeError(f"{what} failed ({rc}): " + L.trba_last_error_string().decode())


Tensor = torch.Tensor
# the raw handle of torch's current stream of a device, without the object around it where torch offers that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = torch.cuda.current_device


def _on(device: torch.device, stream):
    """Context in which `stream` (None: the device's current one) and `device` are current."""
    if stream is None:
        return torch.cuda.device(device)
    if not isinstance(stream, torch.cuda.Stream):
        raise TypeError(f"stream must be a torch.cuda.Stream, got {type(stream).__name__}")
    if stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the tensors are on {device}")
    return torch.cuda.stream(stream)


def _check_tensors(**tensors):
    for name, t in tensors.items():
        if t is not None and not isinstance(t, Tensor):
            raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")


def _check_cuda(name, t, device=None):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _plain(t):
    """t itself, or the values of a view that torch negates or conjugates as it is read."""
    return t.resolve_conj().resolve_neg() if t.is_neg() or t.is_conj() else t


@functools.lru_cache(maxsize=256)
def _select_workspace(code, lines, beams, vocab, device_index):
    return lib().trba_beam_select_workspace(code, lines, beams, vocab)


def _check_beams(beams):
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"1 to {MAX_BEAMS} beams are supported, got {beams}")


def _check_out(name, t, shape, dtype, device):
    _check_tensors(**{name: t})
    _check_cuda(name, t, device)
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous() or t.is_neg():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got {t.dtype} "
                         f"{tuple(t.shape)}")


_IN_PLACE = {("out.scores", "scores"), ("out.finished", "finished")}


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor | None = None, *, eos: int = -1,
                out: BeamStep | None = None, stream=None) -> BeamStep:
    """The best `beams` continuations of every line by running score plus log
    softmax of the logits, best first, ties to the lowest (beam, token).

    logits [lines * beams, vocab] or [lines, beams, vocab], float32, bfloat16
    or float16, any row stride; scores [lines, beams] float32, -inf for a dead
    beam; finished [lines, beams] bool or uint8, or None.  A finished beam
    continues with `eos` at an unchanged score.  A line with too few
    continuations above -inf fills up with score -inf, token eos, parent = the
    slot.  A NaN logit counts as -inf.  `out`: buffers to write into, apart
    from each other and the inputs; its scores and finished may be exactly the
    inputs'."""
    if not (isinstance(scores, Tensor) and isinstance(logits, Tensor)
            and (finished is None or isinstance(finished, Tensor))):
        _check_tensors(scores=scores, logits=logits, finished=finished)
    code = DTYPE_CODES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if scores.dim() != 2 or scores.dtype != torch.float32:
        raise ValueError("scores must be a float32 tensor [lines, beams]")
    lines, beams = scores.shape
    _check_beams(beams)
    shape, strides = logits.shape, logits.stride()
    vocab = shape[-1] if shape else 0
    if len(shape) == 2 and shape[0] == lines * beams:
        ld = strides[0]
    elif len(shape) == 3 and shape[0] == lines and shape[1] == beams:
        if lines > 1 and beams > 1 and strides[0] != beams * strides[1]:
            raise ValueError("logits must have one stride over all (line, beam) rows")
        ld = strides[1] if beams > 1 else strides[0]
    else:
        raise ValueError(f"logits {tuple(shape)} do not fit scores {tuple(scores.shape)}: [lines * beams, vocab] or "
                         "[lines, beams, vocab] is expected")
    if not 1 <= vocab <= 1 << 30 or beams * vocab >= 1 << 31:
        raise ValueError("vocab must be 1 to 2**30 and beams * vocab below 2**31")
    if lines * beams >= 1 << 24:
        raise ValueError("lines * beams must be below 2**24")
    if vocab > 1 and strides[-1] != 1:
        raise ValueError("the logits of a row must be contiguous")
    if lines * beams <= 1:
        ld = vocab
    elif ld < vocab:
        raise ValueError("logits rows overlap")
    if not -1 <= eos < vocab:
        raise ValueError(f"eos must be -1 or in [0, {vocab}), got {eos}")
    device = scores.device
    if finished is not None:
        if eos < 0:
            raise ValueError("finished beams need an end token (eos)")
        if finished.shape != scores.shape or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError("finished must be a bool or uint8 tensor [lines, beams]")
        if finished.device != device:
            _check_cuda("finished", finished, device)
    if not scores.is_cuda or logits.device != device:
        _check_cuda("scores", scores)
        _check_cuda("logits", logits, device)
    if stream is not None or device.index != _current_device():
        with _on(device, stream):
            return beam_select(logits, scores, finished, eos=eos, out=out)
    if logits.is_neg():  # (the copy's strides are others)
        return beam_select(_plain(logits), scores, finished, eos=eos, out=out)
    if scores.is_neg():
        scores = _plain(scores)
    if not scores.is_contiguous():
        scores = scores.contiguous()
    if finished is not None and not finished.is_contiguous():
        finished = finished.contiguous()
    if out is None:
        empty = torch.empty_like
        out = BeamStep(empty(scores), empty(scores, dtype=torch.int32), empty(scores, dtype=torch.int32),
                       empty(scores, dtype=torch.bool))
    else:
        out = BeamStep(*out)
        for name, t, dtype in zip(out._fields, out, (torch.float32, torch.int32, torch.int32, torch.bool)):
            _check_out(f"out.{name}", t, (lines, beams), dtype, device)
        read = {"logits": logits, "scores": scores}
        if finished is not None:
            read["finished"] = finished
        _check_apart({f"out.{n}": t for n, t in zip(out._fields, out)}, read, _IN_PLACE)
    if lines:
        L = lib()
        need = _select_workspace(code, lines, beams, vocab, device.index)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        rc = L.trba_beam_select(logits.data_ptr(), code, ld, scores.data_ptr(),
                                None if finished is None else finished.data_ptr(), lines, beams, vocab, eos,
                                out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
                                work.data_ptr() if need else None, need, _raw_stream(device.index))
        if rc:
            _fail(L, "beam_select", rc)
    return out


def _collapse(shape, src, dst, size):
    """(count, src stride, dst stride) triples, in bytes, outermost first, with
    neighbours merged where both tensors walk on without a gap."""
    dims = []
    for n, a, b in zip(shape, src, dst):
        if n == 1:
            continue
        a, b = a * size, b * size
        if dims and dims[-1][1] == n * a and dims[-1][2] == n * b:
            dims[-1] = (dims[-1][0] * n, a, b)
        else:
            dims.append((n, a, b))
    return dims


def _state(src, dst, dim):
    """The fields of a trba_beam_state for one tensor and its output."""
    size, shape = src.element_size(), src.shape
    if src.is_contiguous() and dst.is_contiguous():
        row, outer = math.prod(shape[dim + 1:]) * size, math.prod(shape[:dim])
        across = shape[dim] * row if outer > 1 else 0
        return src.data_ptr(), dst.data_ptr(), row, row, row, 1, 0, 0, outer, across, across
    outer = _collapse(shape[:dim], src.stride()[:dim], dst.stride()[:dim], size)
    inner = _collapse(shape[dim + 1:], src.stride()[dim + 1:], dst.stride()[dim + 1:], size)
    nbytes = size
    if inner and inner[-1][1] == size and inner[-1][2] == size:
        nbytes *= inner.pop()[0]
    if len(outer) > 1 or len(inner) > 1:
        raise ValueError(f"state of shape {tuple(shape)} and strides {src.stride()}: at most one gap before and one "
                         "after the beam dimension are supported; make it contiguous")
    o, om = outer[0] if outer else (1, 0, 0), inner[0] if inner else (1, 0, 0)
    if ((nbytes - 1) // 1024 + 1) * om[0] * o[0] * shape[dim] > MOST_PARTS:
        raise ValueError(f"state of shape {tuple(shape)} and strides {src.stride()} is too large: its rows fall into "
                         f"more than {MOST_PARTS} contiguous parts")
    return (src.data_ptr(), dst.data_ptr(), nbytes, src.stride(dim) * size, dst.stride(dim) * size, *om, *o)


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, *, dim: int = 0,
                 out: Sequence[torch.Tensor] | None = None, stream=None) -> list[torch.Tensor]:
    """Row (l, k) of every state becomes row (l, parents[l, k]).

    states: tensors of any type whose dimension `dim` is lines * beams, for
    instance h and c [lines * beams, hidden], stacked layers [layers, lines *
    beams, hidden] (dim=1) or the filled part of a cache, cache[:, :, :n];
    parents [lines, beams] int32 as beam_select returns them.  Returns new
    tensors, or writes into `out` (the same shapes and types, apart from the
    states and each other: keep two sets and use them in turn)."""
    states = list(states)
    if not (isinstance(parents, Tensor) and all(isinstance(t, Tensor) for t in states)):
        _check_tensors(parents=parents, **{f"states[{i}]": t for i, t in enumerate(states)})
    if parents.dim() != 2 or parents.dtype != torch.int32:
        raise ValueError("parents must be an int32 tensor [lines, beams]")
    lines, beams = parents.shape
    _check_beams(beams)
    rows = lines * beams
    if rows >= 1 << 24:
        raise ValueError("lines * beams must be below 2**24")
    device = parents.device
    elsewhere, lazy = False, parents.is_neg()
    for i, t in enumerate(states):
        n = t.dim()
        if not -n <= dim < n:
            raise ValueError(f"states[{i}] has no dimension {dim}")
        if t.shape[dim] != rows:
            raise ValueError(f"states[{i}]: dimension {dim} is {t.shape[dim]}, expected lines * beams = {rows}")
        if t.device != device:
            elsewhere = True
        if t.is_neg() or t.is_conj():
            lazy = True
    if out is not None:
        out = list(out)
        if len(out) != len(states):
            raise ValueError(f"out has {len(out)} tensors for {len(states)} states")
        for i, (t, o) in enumerate(zip(states, out)):
            _check_tensors(**{f"out[{i}]": o})
            if o.shape != t.shape or o.dtype != t.dtype:
                raise ValueError(f"out[{i}] must have the shape and type of states[{i}]")
            if o.is_neg() or o.is_conj():
                raise ValueError(f"out[{i}] is a negated or conjugated view")
        _check_apart({f"out[{i}]": o for i, o in enumerate(out)},
                     {"parents": parents, **{f"states[{i}]": t for i, t in enumerate(states)}})
        for i, o in enumerate(out):
            _check_cuda(f"out[{i}]", o, device)
    if not parents.is_cuda:
        _check_cuda("parents", parents)
    if elsewhere:
        for i, t in enumerate(states):
            _check_cuda(f"states[{i}]", t, device)
    if stream is not None or device.index != _current_device():
        with _on(device, stream):
            return beam_reorder(states, parents, dim=dim, out=out)
    if lazy:
        parents, states = _plain(parents), [_plain(t) for t in states]
    if not parents.is_contiguous():
        parents = parents.contiguous()
    if out is None:
        out = [torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=device)
               for t in states]
    fields = []
    for t, o in zip(states, out):
        if t.numel():
            fields += _state(t, o, dim if dim >= 0 else dim + t.dim())
    if fields:
        L = lib()
        rc = L.trba_beam_reorder(struct.pack(f"={len(fields)}q", *fields), len(fields) // 11, parents.data_ptr(),
                                 lines, beams, _raw_stream(device.index))
        if rc:
            _fail(L, "beam_reorder", rc)
    return out


def _span(t):
    """First and one-past-last byte that a tensor's elements reach."""
    last = sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _interleaved(a, b):
    """Whether two tensors share no byte although their ranges of memory do:
    both lie side by side within every period of a stride that they have in
    common (halves of the same wider rows, for instance)."""
    dims = [[(n - 1, st * t.element_size()) for n, st in zip(t.shape, t.stride()) if n > 1] for t in (a, b)]
    apart = b.data_ptr() - a.data_ptr()
    for period in {st for _, st in dims[0]} & {st for _, st in dims[1]} - {0}:
        wide = [t.element_size() + sum(n * st for n, st in d if st % period) for t, d in zip((a, b), dims)]
        if apart % period >= wide[0] and -apart % period >= wide[1]:
            return True
    return False


def _check_apart(written, read, same=()):
    """Refuses outputs that share memory with themselves, each other or an
    input; `same`: (output, input) names that may be one buffer."""
    spans = []
    for group, is_out in ((written, True), (read, False)):
        for name, t in group.items():
            n = t.numel()
            if not n:
                continue
            if t.is_contiguous():
                lo = t.data_ptr()
                spans.append((lo, lo + n * t.element_size(), is_out, name, t))
                continue
            if is_out:
                reach = 1
                for st, m in sorted(zip(t.stride(), t.shape)):
                    if m > 1 and st < reach:
                        raise ValueError(f"{name} is a broadcast view, or overlaps itself")
                    reach += (m - 1) * st
            spans.append((*_span(t), is_out, name, t))
    spans.sort(key=lambda span: span[:4])
    for i, (lo, hi, is_out, name, t) in enumerate(spans):
        for lo2, hi2, is_out2, name2, t2 in spans[i + 1:]:
            if lo2 >= hi:
                break
            if not (is_out or is_out2):
                continue
            a, b = (name, name2) if is_out else (name2, name)
            if not ((a, b) in same and (lo, hi) == (lo2, hi2)) and not _interleaved(t, t2):
                raise ValueError(f"{a} overlaps {b}")


def beam_sequences(tokens: torch.Tensor, parents: torch.Tensor, *, eos: int = -1, pad: int = 0, out=None,
                   stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(sequences [lines, beams, steps] int32, lengths [lines, beams] int32) of
    the paths that end in the last step's slots, from the [steps, lines,
    beams] int32 tokens and parents of all steps: each path's tokens before
    its first `eos`, then `pad`.  `out`: the two to write into, apart from the
    inputs and each other."""
    if not (isinstance(tokens, Tensor) and isinstance(parents, Tensor)):
        _check_tensors(tokens=tokens, parents=parents)
    if tokens.dim() != 3 or tokens.dtype != torch.int32 or parents.shape != tokens.shape or parents.dtype != torch.int32:
        raise ValueError("tokens and parents must be int32 tensors [steps, lines, beams]")
    steps, lines, beams = tokens.shape
    _check_beams(beams)
    if lines * beams >= 1 << 24 or steps >= 1 << 24:
        raise ValueError("lines * beams and steps must be below 2**24")
    for name, v in (("eos", eos), ("pad", pad)):
        if not -2 ** 31 <= v < 2 ** 31:
            raise ValueError(f"{name} must fit in 32 bits, got {v}")
    device = tokens.device
    _check_cuda("tokens", tokens)
    _check_cuda("parents", parents, device)
    if stream is not None or device.index != _current_device():
        with _on(device, stream):
            return beam_sequences(tokens, parents, eos=eos, pad=pad, out=out)
    if tokens.is_neg() or parents.is_neg():
        tokens, parents = _plain(tokens), _plain(parents)
    tokens, parents = tokens.contiguous(), parents.contiguous()
    if out is None:
        out = (torch.empty((lines, beams, steps), dtype=torch.int32, device=device),
               torch.empty((lines, beams), dtype=torch.int32, device=device))
    else:
        seq, lengths = out
        _check_out("out[0]", seq, (lines, beams, steps), torch.int32, device)
        _check_out("out[1]", lengths, (lines, beams), torch.int32, device)
        _check_apart({"out[0]": seq, "out[1]": lengths}, {"tokens": tokens, "parents": parents})
        out = (seq, lengths)
    if lines:
        L = lib()
        rc = L.trba_beam_sequences(tokens.data_ptr(), parents.data_ptr(), steps, lines, beams, eos, pad,
                                   out[0].data_ptr(), out[1].data_ptr(), _raw_stream(device.index))
        if rc:
            _fail(L, "beam_sequences", rc)
    return out
