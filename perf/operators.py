"""Cases of the decoding operators: beam search (selection, reordering of the
states, tracing back the sequences) and the 4-bit linear layer that a serving
decoder reads its weights through.

Each case is measured twice on the same inputs: in its plain form (elementary
torch operations, below) and through the framework's entry points
(trba_b200.decode, trba_b200.ops.LinearInt4).
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

NEG = float("-inf")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}


def _package():
    """This repository's package; its folder name is not an identifier."""
    name = "trba_b200"
    if name not in sys.modules:
        pkg = Path(__file__).resolve().parent.parent / "trba-rust_b200"
        spec = importlib.util.spec_from_file_location(name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    from trba_b200 import decode, ops
    return decode, ops


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # one handwritten line, 5 beams over the recogniser's 130 classes: pure latency
        dict(name="select_line", op="select", lines=1, beams=5, vocab=130, dtype="f32", first=False, masked=False),
        # the benchmark's batch of 512 lines, first decoding step (one live beam a line)
        dict(name="select_batch", op="select", lines=512, beams=5, vocab=130, dtype="f32", first=True, masked=False),
        # word-piece vocabulary of odd size in bf16 (rows start at odd addresses), a lexicon masks most of it
        dict(name="select_lexicon", op="select", lines=48, beams=8, vocab=50001, dtype="bf16", first=False, masked=True),
        # the largest selection: f32 logits of a 64 Ki vocabulary, 10 beams on 64 lines
        dict(name="select_large", op="select", lines=64, beams=10, vocab=65536, dtype="f32", first=False, masked=True),
        # the attention decoder's h and c of one line
        dict(name="reorder_line", op="reorder", lines=1, beams=5, kind="state", tensors=2, width=64, heads=1, length=1,
             room=1, dtype="f32"),
        # stacked LSTM states [layers, lines * beams, hidden] of a large batch, odd width
        dict(name="reorder_layers", op="reorder", lines=512, beams=5, kind="layers", tensors=4, width=255, heads=2,
             length=1, room=1, dtype="f32"),
        # key and value caches of 4 layers, the filled part (odd) of the room that was allocated
        dict(name="reorder_cache", op="reorder", lines=32, beams=8, kind="cache", tensors=8, width=64, heads=8,
             length=333, room=512, dtype="bf16"),
        # sequences of the benchmark's batch: 21 steps
        dict(name="trace_batch", op="trace", lines=512, beams=5, steps=21),
        # a long page transcript: one dependent walk of 2000 steps a beam
        dict(name="trace_long", op="trace", lines=16, beams=16, steps=2000),
        # one line's LSTM gates, 4 * 256 rows over [input, hidden] = 512
        dict(name="linear_gates", op="linear", rows=1, outs=1024, ins=512, group=64, dtype="f32", scales="f32"),
        # a single token through a layer larger than the L2 cache
        dict(name="linear_token", op="linear", rows=1, outs=16384, ins=16384, group=128, dtype="bf16", scales="f16"),
        # 8 lines of 5 beams into an odd vocabulary from an odd width
        dict(name="linear_beams", op="linear", rows=40, outs=50001, ins=4099, group=32, dtype="f16", scales="f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["select", "reorder", "trace", "linear", "select", "linear"])
    if op == "select":
        beams, lines = _log(rng, 1, 32), _log(rng, 1, 512)
        vocab = _log(rng, 100, max(101, min(131072, 64 * 10 * 65536 // (lines * beams))))
        return dict(op=op, lines=lines, beams=beams, vocab=max(vocab, beams), dtype=rng.choice(["f32", "bf16", "f16"]),
                    first=rng.random() < 0.25, masked=rng.random() < 0.5)
    if op == "reorder":
        lines, beams, kind = _log(rng, 1, 512), _log(rng, 1, 32), rng.choice(["state", "layers", "cache"])
        tensors, dtype = rng.randint(1, 12), rng.choice(["f32", "bf16", "f16", "i8"])
        heads = 1 if kind == "state" else rng.randint(1, 8)
        width = _log(rng, 16, 128) if kind == "cache" else _log(rng, 32, 2048)
        most = 32 * 8 * 8 * 8 * 333 * 64 * 2 // (lines * beams * tensors * heads * width * SIZE[dtype])
        length = _log(rng, 1, max(1, min(1000, most))) if kind == "cache" else 1
        if most < 1:
            tensors, width = 1, 64
        return dict(op=op, lines=lines, beams=beams, kind=kind, tensors=tensors, width=width, heads=heads,
                    length=length, room=length + (rng.randint(0, length) if kind == "cache" else 0), dtype=dtype)
    if op == "trace":
        beams, steps = _log(rng, 1, 32), _log(rng, 1, 2000)
        return dict(op=op, lines=_log(rng, 1, max(1, min(512, 16 * 16 * 2000 // (beams * steps)))), beams=beams,
                    steps=steps)
    rows, ins = _log(rng, 1, 64), _log(rng, 64, 16384)
    outs = _log(rng, 64, min(65536, 16384 * 14000 // ins, 8 * 10 ** 9 // (ins * rows)))
    return dict(op=op, rows=rows, outs=outs, ins=ins, group=rng.choice([32, 64, 128]),
                dtype=rng.choice(["f32", "bf16", "f16"]), scales=rng.choice(["f32", "f16"]))


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _inputs(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def ints(hi, *shape, dtype=torch.int32):
        return torch.randint(0, hi, shape, generator=g, device=dev, dtype=dtype)

    op = case["op"]
    if op == "select":
        L, K, V = case["lines"], case["beams"], case["vocab"]
        x = randn(L * K, V).mul_(3.0).to(DTYPES[case["dtype"]])
        eos = 2
        if case["masked"]:  # a lexicon leaves a fifth of the tokens, on one line of the batch nothing
            allowed = torch.rand(L, V, generator=g, device=dev) < 0.2
            if L > 4:
                allowed[L // 2] = False
            x.view(L, K, V).masked_fill_(~allowed[:, None, :], NEG)
        scores = randn(L, K).abs_().mul_(2.0).cumsum(1).neg_()
        done = torch.rand(L, K, generator=g, device=dev) < 0.2
        if case["first"]:
            scores.fill_(NEG)[:, 0] = 0.0
            done.fill_(False)
        return dict(logits=x, scores=scores, finished=done, eos=eos)
    if op == "reorder":
        L, K, W, dtype = case["lines"], case["beams"], case["width"], DTYPES[case["dtype"]]
        shape = {"state": (L * K, W), "layers": (case["heads"], L * K, W),
                 "cache": (L * K, case["heads"], case["room"], W)}[case["kind"]]
        make = (lambda: ints(255, *shape, dtype=torch.int16).sub_(127).to(dtype)) if dtype == torch.int8 else (
            lambda: randn(*shape).to(dtype))
        return dict(states=[make() for _ in range(case["tensors"])], parents=ints(K, L, K),
                    dim=1 if case["kind"] == "layers" else 0, length=case["length"], cache=case["kind"] == "cache")
    if op == "trace":
        T, L, K = case["steps"], case["lines"], case["beams"]
        tokens, parents = ints(130, T, L, K).clamp_(min=3), ints(K, T, L, K)
        ends = ints(2 * T, L, K)  # half of the beams reach the end token, which then repeats
        tokens.masked_fill_(torch.arange(T, device=dev)[:, None, None] >= ends, 2)
        return dict(tokens=tokens, parents=parents, eos=2, pad=0)
    M, N, K, G = case["rows"], case["outs"], case["ins"], case["group"]
    x = randn(M, K)
    x[:, :: max(1, K // 7)] *= 20.0  # a few channels are far larger than the others
    scales = randn(N, -(-K // G)).abs_().add_(0.1).mul_(0.02)
    return dict(x=x.to(DTYPES[case["dtype"]]), codes=ints(256, N, -(-K // 2), dtype=torch.uint8),
                scales=scales.to(DTYPES[case["scales"]]), bias=randn(N), ins=K, group=G)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["op"] = case["op"]
    if own:
        decode, ops = _package()
        if case["op"] == "linear":  # the layer a serving program holds
            state["layer"] = ops.LinearInt4.from_codes(state["codes"], state["scales"], in_features=state["ins"],
                                                       group=state["group"], bias=state["bias"])
            state["call"] = state["layer"].forward
        else:
            state["call"] = {"select": decode.beam_select, "reorder": decode.beam_reorder,
                             "trace": decode.beam_sequences}[case["op"]]
    return state


# --------------------------------------------------------------------- run --
def run(s):
    if s["op"] == "select":
        if own:
            return tuple(s["call"](s["logits"], s["scores"], s["finished"], eos=s["eos"]))
        return plain_select(s["logits"], s["scores"], s["finished"], s["eos"])
    if s["op"] == "reorder":
        states = [t[:, :, :s["length"]] for t in s["states"]] if s["cache"] else s["states"]
        if own:
            return s["call"](states, s["parents"], dim=s["dim"])
        return plain_reorder(states, s["parents"], s["dim"])
    if s["op"] == "trace":
        if own:
            return tuple(s["call"](s["tokens"], s["parents"], eos=s["eos"], pad=s["pad"]))
        return plain_sequences(s["tokens"], s["parents"], s["eos"], s["pad"])
    if own:
        return s["call"](s["x"])
    return plain_linear(s["x"], s["codes"], s["scales"], s["bias"], s["ins"], s["group"])


def plain_select(logits, scores, finished, eos):
    """One step of beam search: the best `beams` of scores[b] + log softmax(logits[b, v]) over all beams and tokens
    of a line; a finished beam goes on with the end token alone and keeps its score.  In 64 bits: neighbours in the
    order may differ by less than 32 bits hold.  Ties go to the lowest (beam, token)."""
    L, K = scores.shape
    V = logits.shape[-1]
    x = logits.reshape(L, K, V).double()
    x = torch.where(torch.isnan(x), NEG, x)
    top = x.amax(-1, keepdim=True)
    z = torch.where(x == top, 0.0, x - top)
    z = torch.where(x == NEG, NEG, z)
    total = scores.double()[:, :, None] + (z - z.exp().sum(-1, keepdim=True).log())
    only = torch.full_like(total, NEG)
    only[:, :, eos] = scores.double()
    total = torch.where(finished[:, :, None], only, total).reshape(L, K * V)
    total = torch.where(total.float() > NEG, total, NEG)  # NaN too
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    dead = best == NEG
    slot = torch.arange(K, device=x.device).expand(L, K)
    parents = torch.where(dead, slot, at // V)
    tokens = torch.where(dead, eos, at % V)
    done = dead | (tokens == eos) | finished.gather(1, parents)
    return best.float(), tokens.int(), parents.int(), done


def plain_reorder(states, parents, dim):
    """Row (line, k) of every state becomes row (line, parents[line, k])."""
    L, K = parents.shape
    rows = (torch.arange(L, device=parents.device)[:, None] * K + parents).reshape(-1)
    return [t.index_select(dim, rows) for t in states]


def plain_sequences(tokens, parents, eos, pad):
    """The token sequences that end in the last step's slots: slot[t - 1] = parents[t][slot[t]], composed by doubling."""
    T, L, K = tokens.shape
    device = tokens.device
    last = torch.arange(K, device=device).expand(1, L, K)
    slot = torch.cat([parents[1:].long(), last])
    step = 1
    while step < T:
        slot = torch.cat([slot[:-step].gather(2, slot[step:]), slot[-step:]])
        step *= 2
    seq = tokens.gather(2, slot).permute(1, 2, 0)
    over = (seq == eos).int().cumsum(2) > 0
    return torch.where(over, pad, seq).int(), (T - over.sum(2)).int()


def plain_linear(x, codes, scales, bias, ins, group):
    """x [rows, ins] times the weights (code - 8) * scale, two codes a byte (the even column's in the low half)."""
    N = codes.shape[0]
    q = torch.stack([codes & 15, codes >> 4], -1).reshape(N, -1)[:, :ins].float() - 8.0
    w = q * scales.float().repeat_interleave(group, 1)[:, :ins]
    return (x.float() @ w.T + bias).to(x.dtype)


def work(case):
    op = case["op"]
    if op == "select":
        rows = case["lines"] * case["beams"]
        # dead and finished beams' logits are not needed: about a fifth of the beams are finished after the first step
        n = (case["lines"] if case["first"] else 0.8 * rows) * case["vocab"]
        return dict(bytes=n * SIZE[case["dtype"]] + rows * 18, flops=4 * n)
    if op == "reorder":
        n = case["lines"] * case["beams"] * case["tensors"] * case["width"] * case["heads"] * case["length"]
        return dict(bytes=2 * n * SIZE[case["dtype"]] + case["lines"] * case["beams"] * 4, flops=0)
    if op == "trace":
        n = case["lines"] * case["beams"]
        return dict(bytes=12 * n * case["steps"] + 4 * n, flops=0)
    M, N, K = case["rows"], case["outs"], case["ins"]
    return dict(bytes=N * -(-K // 2) + N * -(-K // case["group"]) * SIZE[case["scales"]] + 4 * N
                + M * (N + K) * SIZE[case["dtype"]], flops=2 * M * N * K)


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    if case["op"] in ("reorder", "trace"):
        return None  # copies and whole numbers: nothing is computed that could be rounded
    s = {k: v.double().cpu().numpy() if torch.is_tensor(v) and v.is_floating_point() else v
         for k, v in _inputs(case, seed).items()}
    if case["op"] == "linear":
        codes, N, K, G = s["codes"].cpu().numpy(), case["outs"], case["ins"], case["group"]
        if case["rows"] * N * K > 2e10:
            return None
        y = np.empty((case["rows"], N))
        at = np.arange(K)
        for lo in range(0, N, 2048):
            hi = min(N, lo + 2048)
            half = codes[lo:hi, at // 2]
            q = np.where(at % 2 == 0, half % 16, half // 16).astype(np.float64) - 8
            y[:, lo:hi] = s["x"] @ (q * s["scales"][lo:hi, at // G]).T + s["bias"][lo:hi]
        return y
    L, K, V = case["lines"], case["beams"], case["vocab"]
    done, eos = s["finished"].cpu().numpy(), s["eos"]
    logits = s["logits"].reshape(L, K, V)
    out = np.empty((L, K)), np.empty((L, K), np.int32), np.empty((L, K), np.int32), np.empty((L, K), bool)
    for b in range(L):
        found = []  # (score, beam, token) of each beam's best
        for k in range(K):
            run_score = s["scores"][b, k]
            if run_score == NEG:
                continue
            if done[b, k]:
                found.append((-run_score, k, eos))
                continue
            row = logits[b, k]
            m = row.max()
            if m == NEG:
                continue
            logp = row - (m + np.log(np.exp(row - m).sum()))
            near = np.argpartition(-logp, K - 1)[:K] if V > K else np.arange(V)
            near = np.flatnonzero(logp >= logp[near].min())
            found += [(-(run_score + logp[v]), k, int(v)) for v in near if logp[v] > NEG]
        found.sort()
        for k in range(K):
            score, parent, token = found[k] if k < len(found) else (math.inf, k, eos)
            out[0][b, k], out[1][b, k], out[2][b, k] = -score, token, parent
            out[3][b, k] = token == eos or bool(done[b, parent])
    return out
