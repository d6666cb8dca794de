// Beam-search operators (include/trba_decode.h): selection of the best (beam,
// token) pairs, reordering of the beams' states, token sequences from the
// history.  No counterpart in the reference, whose decoder is greedy
// (src/attn.rs:368-447).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "trba_decode.h"

namespace trba {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kNone = 0x7fffffff;

// -------------------------------------------------------------- selection --
template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32(__half v) {
    return __half2float(v);
}

// The best entries of a warp, one a lane, best first: larger value, then lower
// index.  Lanes that hold no entry have (-inf, kNone).
struct WarpList {
    float v = -INFINITY;
    int i = kNone;
    // Inserts (x, at), the same in every lane, if it is among the best `k`.
    __device__ __forceinline__ void insert(float x, int at, int lane) {
        const int pos = __popc(__ballot_sync(kFull, v > x || (v == x && i < at)));
        const float pv = __shfl_up_sync(kFull, v, 1);
        const int pi = __shfl_up_sync(kFull, i, 1);
        if (lane == pos) {
            v = x;
            i = at;
        } else if (lane > pos) {
            v = pv;
            i = pi;
        }
    }
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

constexpr int kSelThreads = 256;

// One CTA a line, a warp a beam at a time: the row's best `beams` tokens (the
// order within a row is that of the logits) and its log sum of exponentials;
// then one warp merges the beams' lists, its lane b at the head of beam b's.
template <class T>
__global__ void __launch_bounds__(kSelThreads) beam_select_kernel(
    const T *__restrict__ logits, i64 ld, const float *scores, const uint8_t *finished, int beams, int vocab, int eos,
    float *out_scores, int32_t *__restrict__ out_tokens, int32_t *__restrict__ out_parents, uint8_t *out_finished) {
    __shared__ double s_score[TRBA_MAX_BEAMS][TRBA_MAX_BEAMS];
    __shared__ int s_tok[TRBA_MAX_BEAMS][TRBA_MAX_BEAMS];
    __shared__ uint8_t s_fin[TRBA_MAX_BEAMS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const i64 slot0 = (i64)blockIdx.x * beams;
    for (int b = warp; b < beams; b += kSelThreads / 32) {
        const float sc = scores[slot0 + b];
        const bool fin = finished && finished[slot0 + b];
        const bool dead = !(sc > -INFINITY);
        double out = -INFINITY;
        int tok = kNone;
        if (fin && !dead) {
            if (lane == 0) {
                out = (double)sc;
                tok = eos;
            }
        } else if (!dead) {
            const T *row = logits + (slot0 + b) * ld;
            WarpList best;
            float thr = -INFINITY, m = -INFINITY;
            double sum = 0.0;
            for (int c0 = 0; c0 < vocab; c0 += 32) {
                const int c = c0 + lane;
                const float x = fmaxf(c < vocab ? to_f32(row[c]) : -INFINITY, -INFINITY);  // NaN counts as -inf
                if (x > -INFINITY) {
                    if (x > m) {
                        sum = sum * (double)__expf(m - x) + 1.0;
                        m = x;
                    } else {
                        sum += x == m ? 1.0 : (double)__expf(x - m);
                    }
                }
                // candidates in index order: a later one that ties with the last of the list loses
                unsigned some = __ballot_sync(kFull, x > thr);
                while (some) {
                    const int src = __ffs(some) - 1;
                    best.insert(__shfl_sync(kFull, x, src), c0 + src, lane);
                    thr = __shfl_sync(kFull, best.v, beams - 1);
                    some &= some - 1;
                    some &= __ballot_sync(kFull, x > thr);
                }
            }
            const float top = warp_max(m);
            const double lse = log(warp_sum(m > -INFINITY ? (m == top ? sum : sum * exp((double)m - (double)top)) : 0.0));
            if (lane < beams && best.i != kNone) {
                out = (double)sc + ((best.v == top ? 0.0 : (double)best.v - (double)top) - lse);
                tok = best.i;
            }
        }
        if (!((float)out > -INFINITY)) out = -INFINITY;
        if (lane < beams) {
            s_score[b][lane] = out;
            s_tok[b][lane] = tok;
        }
        if (lane == 0) s_fin[b] = fin;
    }
    __syncthreads();
    if (warp != 0) return;
    int head = 0;
    for (int k = 0; k < beams; ++k) {
        double v = lane < beams && head < beams ? s_score[lane][head] : -INFINITY;
        int who = lane;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {  // ties between beams go to the lower beam
            const double ov = __shfl_xor_sync(kFull, v, o);
            const int ow = __shfl_xor_sync(kFull, who, o);
            if (ov > v || (ov == v && ow < who)) {
                v = ov;
                who = ow;
            }
        }
        const bool none = !(v > -INFINITY);
        if (lane == who) {
            const int tok = none ? (eos < 0 ? 0 : eos) : s_tok[who][head];
            const int parent = none ? k : who;
            out_scores[slot0 + k] = (float)v;
            out_tokens[slot0 + k] = tok;
            out_parents[slot0 + k] = parent;
            out_finished[slot0 + k] = eos >= 0 && (none || tok == eos || s_fin[who]);
            ++head;
        }
    }
}

// -------------------------------------------------------------- reordering --
constexpr int kMaxStates = 16;
struct StateView {
    const char *src;
    char *dst;
    i64 units, src_row, dst_row, mid, src_mid, dst_mid, src_outer, dst_outer, total;
    int vec;
};
struct StateViews {
    StateView s[kMaxStates];
};

// Grid y is the state; its units of `vec` bytes in the order [outer][row][mid][unit].
template <class V>
__device__ __forceinline__ void reorder_units(const StateView &s, const int32_t *__restrict__ parents, i64 rows,
                                              int beams) {
    GRID_LOOP(e, s.total) {
        const i64 u = e % s.units, q = e / s.units, mid = q % s.mid, q2 = q / s.mid, row = q2 % rows, o = q2 / rows;
        const int p = parents[row];
        if ((unsigned)p >= (unsigned)beams) continue;
        const i64 from = row - row % beams + p;
        *reinterpret_cast<V *>(s.dst + o * s.dst_outer + row * s.dst_row + mid * s.dst_mid + u * sizeof(V)) =
            *reinterpret_cast<const V *>(s.src + o * s.src_outer + from * s.src_row + mid * s.src_mid + u * sizeof(V));
    }
}

__global__ void __launch_bounds__(256) beam_reorder_kernel(const __grid_constant__ StateViews st,
                                                           const int32_t *__restrict__ parents, i64 rows, int beams) {
    const StateView &s = st.s[blockIdx.y];
    if (s.vec == 16) reorder_units<uint4>(s, parents, rows, beams);
    else if (s.vec == 8) reorder_units<uint2>(s, parents, rows, beams);
    else if (s.vec == 4) reorder_units<uint32_t>(s, parents, rows, beams);
    else if (s.vec == 2) reorder_units<uint16_t>(s, parents, rows, beams);
    else reorder_units<uint8_t>(s, parents, rows, beams);
}

// --------------------------------------------------------------- sequences --
// One thread a slot walks from the last step to the first.
__global__ void __launch_bounds__(128) beam_sequences_kernel(const int32_t *__restrict__ tokens,
                                                             const int32_t *__restrict__ parents, int steps, int lines,
                                                             int beams, int eos, int pad, int32_t *__restrict__ seq,
                                                             int32_t *__restrict__ lengths) {
    const i64 n = (i64)lines * beams, e = (i64)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= n) return;
    const i64 line0 = e - e % beams;
    int slot = (int)(e % beams), len = steps;
    bool bad = false;
    for (int t = steps - 1; t >= 0; --t) {
        const i64 at = t * n + line0 + slot;
        const int tok = tokens[at];
        seq[e * steps + t] = tok;
        if (tok == eos) len = t;
        if (t > 0) {
            slot = parents[at];
            if ((unsigned)slot >= (unsigned)beams) {
                bad = true;
                break;
            }
        }
    }
    for (int t = bad ? 0 : len; t < steps; ++t) seq[e * steps + t] = pad;
    lengths[e] = bad ? -1 : len;
}

int launched() {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
    return (int)e;
}

template <class T>
int select(const void *logits, i64 ld, const float *scores, const uint8_t *finished, int lines, int beams, int vocab,
           int eos, float *out_scores, int32_t *out_tokens, int32_t *out_parents, uint8_t *out_finished,
           cudaStream_t st) {
    beam_select_kernel<T><<<lines, kSelThreads, 0, st>>>(static_cast<const T *>(logits), ld, scores, finished, beams,
                                                         vocab, eos, out_scores, out_tokens, out_parents,
                                                         out_finished);
    return launched();
}

}  // namespace
}  // namespace trba

using namespace trba;

extern "C" {

int trba_beam_select(const void *logits, int dtype, long long ld, const float *scores, const uint8_t *finished,
                     int lines, int beams, int vocab, int eos, float *out_scores, int32_t *out_tokens,
                     int32_t *out_parents, uint8_t *out_finished, void *stream) {
    TRBA_REQUIRE_RET(lines >= 0 && beams > 0 && beams <= TRBA_MAX_BEAMS && vocab > 0 && ld >= vocab &&
                         (i64)beams * vocab < (1ll << 31),
                     "trba_beam_select: bad sizes", -1);
    TRBA_REQUIRE_RET(eos >= -1 && eos < vocab && (eos >= 0 || !finished),
                     "trba_beam_select: eos outside the vocabulary, or finished beams without an end token", -1);
    TRBA_REQUIRE_RET(dtype == TRBA_F32 || dtype == TRBA_BF16 || dtype == TRBA_F16,
                     "trba_beam_select: unknown element type", -1);
    if (lines == 0) return 0;
    TRBA_REQUIRE_RET(logits && scores && out_scores && out_tokens && out_parents && out_finished,
                     "trba_beam_select: null pointer", -1);
    TRBA_REQUIRE_RET(reinterpret_cast<uintptr_t>(logits) % (dtype == TRBA_F32 ? 4 : 2) == 0,
                     "trba_beam_select: logits are not aligned to their elements", -1);
    cudaStream_t st = as_stream(stream);
    if (dtype == TRBA_F32)
        return select<float>(logits, ld, scores, finished, lines, beams, vocab, eos, out_scores, out_tokens,
                             out_parents, out_finished, st);
    if (dtype == TRBA_BF16)
        return select<__nv_bfloat16>(logits, ld, scores, finished, lines, beams, vocab, eos, out_scores, out_tokens,
                                     out_parents, out_finished, st);
    return select<__half>(logits, ld, scores, finished, lines, beams, vocab, eos, out_scores, out_tokens, out_parents,
                          out_finished, st);
}

int trba_beam_reorder(const trba_beam_state *states, int n_states, const int32_t *parents, int lines, int beams,
                      void *stream) {
    TRBA_REQUIRE_RET(n_states >= 0 && lines >= 0 && beams > 0 && beams <= TRBA_MAX_BEAMS,
                     "trba_beam_reorder: bad sizes", -1);
    if (n_states == 0 || lines == 0) return 0;
    TRBA_REQUIRE_RET(states && parents, "trba_beam_reorder: null pointer", -1);
    const i64 rows = (i64)lines * beams;
    for (int i = 0; i < n_states; ++i) {
        const trba_beam_state &s = states[i];
        TRBA_REQUIRE_RET(s.bytes >= 0 && s.mid >= 0 && s.outer >= 0, "trba_beam_reorder: negative size", -1);
        TRBA_REQUIRE_RET((s.src && s.dst) || s.bytes == 0 || s.mid == 0 || s.outer == 0,
                         "trba_beam_reorder: null state", -1);
    }
    for (int i0 = 0; i0 < n_states; i0 += kMaxStates) {
        StateViews v{};
        int n = 0;
        i64 most = 0;
        for (int i = i0; i < n_states && i < i0 + kMaxStates; ++i) {
            const trba_beam_state &s = states[i];
            if (s.bytes == 0 || s.mid == 0 || s.outer == 0) continue;
            // the widest unit that every address of the view is a multiple of
            i64 bits = (i64)reinterpret_cast<uintptr_t>(s.src) | (i64)reinterpret_cast<uintptr_t>(s.dst) | s.bytes |
                       s.src_row | s.dst_row;
            if (s.mid > 1) bits |= s.src_mid | s.dst_mid;
            if (s.outer > 1) bits |= s.src_outer | s.dst_outer;
            int vec = 16;
            while (bits & (vec - 1)) vec >>= 1;
            StateView &d = v.s[n++];
            d.src = static_cast<const char *>(s.src);
            d.dst = static_cast<char *>(s.dst);
            d.vec = vec;
            d.units = s.bytes / vec;
            d.src_row = s.src_row, d.dst_row = s.dst_row;
            d.mid = s.mid, d.src_mid = s.src_mid, d.dst_mid = s.dst_mid;
            d.src_outer = s.src_outer, d.dst_outer = s.dst_outer;
            d.total = d.units * s.mid * s.outer * rows;
            if (d.total > most) most = d.total;
        }
        if (n == 0) continue;
        beam_reorder_kernel<<<dim3(grid_for(most), n), 256, 0, as_stream(stream)>>>(v, parents, rows, beams);
        if (const int e = launched()) return e;
    }
    return 0;
}

int trba_beam_sequences(const int32_t *tokens, const int32_t *parents, int steps, int lines, int beams, int eos,
                        int pad, int32_t *sequences, int32_t *lengths, void *stream) {
    TRBA_REQUIRE_RET(steps >= 0 && lines >= 0 && beams > 0 && beams <= TRBA_MAX_BEAMS &&
                         (i64)lines * beams < (1ll << 31),
                     "trba_beam_sequences: bad sizes", -1);
    if (lines == 0) return 0;
    TRBA_REQUIRE_RET(lengths && (steps == 0 || (tokens && parents && sequences)), "trba_beam_sequences: null pointer",
                     -1);
    const i64 n = (i64)lines * beams;
    beam_sequences_kernel<<<(int)((n + 127) / 128), 128, 0, as_stream(stream)>>>(tokens, parents, steps, lines, beams,
                                                                                 eos, pad, sequences, lengths);
    return launched();
}

}  // extern "C"
