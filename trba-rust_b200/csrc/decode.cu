// Beam-search operators (include/trba_decode.h): selection of the best (beam,
// token) pairs, reordering of the beams' states, token sequences from the
// history.  No counterpart in the reference, whose decoder is greedy
// (src/attn.rs:368-447).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdlib.h>

#include <atomic>
#include <type_traits>

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

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
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
// The value of rank `k` (0: largest) of the warp's 32, by a bitonic sort.
__device__ __forceinline__ float warp_kth(float v, int k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const float w = __shfl_xor_sync(kFull, v, o);
            v = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(v, w) : fminf(v, w);
        }
    return __shfl_sync(kFull, v, k);
}
// Unsigned integers in the order of the floats (no NaN).
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned u = __float_as_uint(v);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned k) {
    return __uint_as_float(k ^ ((unsigned)((int)~k >> 31) | 0x80000000u));
}

// A candidate as one number: the larger value first, then the lower index.
// Values of -inf are no candidates: 0.
typedef unsigned long long Key;
__device__ __forceinline__ Key make_key(float x, int at) {
    return x > -INFINITY ? (Key)ordered(x + 0.0f) << 32 | (unsigned)~at : 0;  // (-0 equals 0)
}
__device__ __forceinline__ float key_value(Key k) { return k ? unordered((unsigned)(k >> 32)) : -INFINITY; }
__device__ __forceinline__ int key_index(Key k) { return (int)~(unsigned)k; }

__device__ __forceinline__ Key exchange(Key v, int o, bool keep_max) {
    const Key w = __shfl_xor_sync(kFull, v, o);
    return (v > w) == keep_max ? v : w;
}
// The warp's 32 keys in descending order, by a bitonic sort; only the first
// `count` lanes have keys.
__device__ __noinline__ Key sort_keys(Key v, int count, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) v = exchange(v, o, ((lane & o) == 0) == ((lane & size) == 0));
        if (count <= size) break;
    }
    return v;
}
// The largest 32 of two descending lists, descending.
__device__ __noinline__ Key merge_keys(Key a, Key b, int lane) {
    const Key r = __shfl_sync(kFull, b, 31 - lane);
    Key v = a > r ? a : r;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = exchange(v, o, (lane & o) == 0);
    return v;
}

// The scan of a row goes in batches of kSelUnroll groups of 16 bytes a lane,
// through a ring of cp.async stages in shared memory.  Rows may start at any
// element: a stage holds the aligned blocks its batch lies in, and a group
// that straddles two is put together from both.  Groups go by their index in
// the row, not by their address, so that equal rows have equal sums wherever
// they start.
constexpr int kSelUnroll = 4, kStages = 2;
constexpr int kStageBytes = kSelUnroll * 512 + 16;
constexpr int kSpans = 16;    // spans of batches whose largest elements are remembered
constexpr int kBuffer = 64;   // candidates kept before they are sorted in
constexpr float kLog2e = 1.4426950408889634f;

// Shared memory of a warp's scan.  The candidates and the list of places to
// look at again use the ring when it is done with, or the spans that a segment
// still in the ring leaves free.
struct __align__(16) Scan {
    uint8_t ring[kStages][kStageBytes];
    float most[kSpans][32];  // the largest element of each lane in each span
    __device__ __forceinline__ Key *cand(bool kept) {  // [kBuffer]
        return kept ? reinterpret_cast<Key *>(most[kStages]) : reinterpret_cast<Key *>(ring);
    }
    __device__ __forceinline__ unsigned short *hit(bool kept) {  // span * 32 + lane, [kSpans * 32]
        return reinterpret_cast<unsigned short *>(cand(kept) + kBuffer);
    }
};
static_assert(kStages * kStageBytes >= kBuffer * 8 + kSpans * 64, "the ring holds candidates and places");
static_assert((kSpans - kStages) * 128 >= kBuffer * 8 + kStages * 64, "so do the spans a short segment leaves free");

// What a warp found in its segment of a row: the largest logit, the sum of
// exp(logit - largest) and its best tokens.
struct Found {
    double sum;
    Key best[TRBA_MAX_BEAMS];
    float top;
};

template <class T>
__device__ __forceinline__ float element(uint32_t w, int half) {
    float v;
    if (sizeof(T) == 4) v = __uint_as_float(w);
    else if (std::is_same<T, __nv_bfloat16>::value) v = __uint_as_float(half ? w & 0xffff0000u : w << 16);
    else v = __half2float(__ushort_as_half((unsigned short)(w >> (16 * half))));
    return v;
}

// Copies the blocks of the elements [base, base + batch) that lie before `end`.
template <class T>
__device__ __forceinline__ void fetch_batch(const T *row, int base, int end, int skew, uint8_t *stage, int lane) {
    const char *src = reinterpret_cast<const char *>(row + base) - skew + lane * 16;
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(stage)) + lane * 16;
    if (base + (kSelUnroll * 32 + 1) * 16 / (int)sizeof(T) <= end) {
#pragma unroll
        for (int u = 0; u < kSelUnroll; ++u)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + u * 512), "l"(src + u * 512) : "memory");
        if (skew && lane == 0)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + kSelUnroll * 512), "l"(src + kSelUnroll * 512)
                         : "memory");
        return;
    }
    // the row's end: the last block only as far as the row goes
#pragma unroll 1
    for (int u = 0; u <= kSelUnroll; ++u) {
        if (u == kSelUnroll && (lane > 0 || skew == 0)) break;
        const int room = (end - base) * (int)sizeof(T) + skew - lane * 16 - u * 512, bytes = min(room, 16);
        if (bytes > 0)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + u * 512), "l"(src + u * 512), "r"(bytes)
                         : "memory");
    }
}

// The elements of +inf of a lane in a batch (they share the row): rare.
template <class T>
__device__ __noinline__ int count_inf(const T *row, int base, int end, int lane) {
    constexpr int N = 16 / sizeof(T);
    int n = 0;
#pragma unroll 1
    for (int k = 0; k < kSelUnroll * N; ++k) {
        const int at = base + (k / N * 32 + lane) * N + k % N;
        if (at < end && to_f32(row[at]) == INFINITY) ++n;
    }
    return n;
}

// Sorts the first 32 candidates of the buffer into the list of the best.
__device__ __forceinline__ Key take_32(Key *cand, Key best, int &count, int lane) {
    __syncwarp();
    Key mine = lane < count ? cand[lane] : 0;
    const Key rest = lane + 32 < count ? cand[lane + 32] : 0;
    __syncwarp();
    if (lane + 32 < count) cand[lane] = rest;
    mine = sort_keys(mine, count, lane);
    count = max(0, count - 32);
    return __any_sync(kFull, best != 0) ? merge_keys(best, mine, lane) : mine;
}
// Appends the lanes' wanted keys to the buffer.
__device__ __forceinline__ void append(Key *cand, Key key, bool want, int &count, int lane) {
    const unsigned some = __ballot_sync(kFull, want);
    if (want) cand[count + __popc(some & ((1u << lane) - 1))] = key;
    count += __popc(some);
}

// Lists the places whose largest element is at least `bar`; returns how many.
__device__ __forceinline__ int list_hits(const Scan &scan, unsigned short *list, int spans, float bar, int lane) {
    const float least = fmaxf(bar, -3.402823466e38f);  // -inf is never one of the best
    int hits = 0;
    __syncwarp();
#pragma unroll 4
    for (int q = 0; q < spans; ++q) {
        const bool hit = scan.most[q][lane] >= least;  // (a lane reads what it wrote itself)
        const unsigned some = __ballot_sync(kFull, hit);
        if (hit) list[hits + __popc(some & ((1u << lane) - 1))] = (unsigned short)(q * 32 + lane);
        hits += __popc(some);
    }
    __syncwarp();
    return hits;
}

// The elements [c0, c1) of a row (c0 a multiple of 32 groups): the sum of
// exp(x - m) under a lane's running largest m, f32 within a batch, f64 beyond,
// and the best `beams`.  The scan itself only remembers each lane's largest
// element of each span of batches.  The beams-th largest of those is a bar
// that at least `beams` elements reach, so only the places whose largest
// reaches it, about as many as there are beams, are looked at again (in the
// ring if the segment still is, else in the cache).
template <class T>
__device__ __forceinline__ void scan_segment(const T *row, int c0, int c1, int beams, int lane, Scan &scan,
                                             Found &out) {
    constexpr int N = 16 / sizeof(T), kBatch = kSelUnroll * 32 * N;
    const int skew = (int)(reinterpret_cast<uintptr_t>(row) & 15);
    const int batches = (c1 - c0 + kBatch - 1) / kBatch, per = (batches + kSpans - 1) / kSpans;
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) {
        if (t < batches) fetch_batch<T>(row, c0 + t * kBatch, c1, skew, scan.ring[t], lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    float m = -INFINITY, most = -INFINITY;
    double sum = 0.0;
    int spans = 0, in_span = 0;
#pragma unroll 1
    for (int t = 0; t < batches; ++t) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        if (t + kStages - 1 < batches)
            fetch_batch<T>(row, c0 + (t + kStages - 1) * kBatch, c1, skew, scan.ring[(t + kStages - 1) % kStages], lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const int base = c0 + t * kBatch;
        float x[kSelUnroll][N];
#pragma unroll
        for (int u = 0; u < kSelUnroll; ++u) {
            const uint4 *q = reinterpret_cast<const uint4 *>(scan.ring[t % kStages]) + u * 32 + lane;
            const uint4 lo = q[0];
            uint32_t w[4] = {lo.x, lo.y, lo.z, lo.w};
            if (skew) {
                const uint4 hi = q[1];
                const uint32_t all[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                const int by = skew >> 2, sh = (skew & 2) * 8;
                uint32_t s[5];
#pragma unroll
                for (int i = 0; i < 5; ++i) {
                    const uint32_t a = by & 1 ? all[i + 1] : all[i], b = by & 1 ? all[min(i + 3, 7)] : all[i + 2];
                    s[i] = by & 2 ? b : a;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(s[i], s[i + 1], sh);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) x[u][e] = element<T>(w[e * (int)sizeof(T) / 4], e & 1);
        }
        if (base + kBatch > c1) {  // the row's last batch
#pragma unroll
            for (int u = 0; u < kSelUnroll; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (base + (u * 32 + lane) * N + e >= c1) x[u][e] = -INFINITY;
        }
        float all = -INFINITY;  // (of a number and a NaN the number is the larger)
#pragma unroll
        for (int u = 0; u < kSelUnroll; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) all = fmaxf(all, x[u][e]);
        if (all > m) {
            sum *= (double)exp2_approx((m - all) * kLog2e);  // 0 while m is -inf (and so is the sum)
            m = all;
        }
        most = fmaxf(most, all);
        if (++in_span == per || t + 1 == batches) {
            scan.most[spans++][lane] = most;
            most = -INFINITY;
            in_span = 0;
        }
        if (m == INFINITY) {
            sum += (double)count_inf<T>(row, base, c1, lane);
        } else if (m > -INFINITY) {
            float part[kSelUnroll];
            bool again = true;
            while (again) {
#pragma unroll
                for (int u = 0; u < kSelUnroll; ++u) {
                    float y[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] = exp2_approx((x[u][e] - m) * kLog2e);
#pragma unroll
                    for (int o = N / 2; o > 0; o >>= 1)
#pragma unroll
                        for (int e = 0; e < o; ++e) y[e] += y[e + o];
                    part[u] = y[0];
                }
                part[0] = (part[0] + part[1]) + (part[2] + part[3]);
                again = part[0] != part[0];
                if (again) {  // NaN counts as -inf
#pragma unroll
                    for (int u = 0; u < kSelUnroll; ++u)
#pragma unroll
                        for (int e = 0; e < N; ++e) x[u][e] = fmaxf(x[u][e], -INFINITY);
                }
            }
            sum += (double)part[0];
        }
    }

    // the bar: first from the lanes' maxima; where that leaves many places, from theirs
    const bool kept = batches <= kStages;
    Key *cand = scan.cand(kept);
    unsigned short *hit = scan.hit(kept);
    float bar = warp_kth(m, beams - 1, lane);
    int hits = list_hits(scan, hit, spans, bar, lane), count = 0;
    Key best = 0;
    if (hits > 32) {
#pragma unroll 1
        for (int h0 = 0; h0 < hits; h0 += 32) {
            Key c = 0;
            if (h0 + lane < hits) {
                const int h = hit[h0 + lane];
                c = make_key(scan.most[h >> 5][h & 31], h0 + lane);
            }
            if (__any_sync(kFull, c > __shfl_sync(kFull, best, beams - 1)))
                best = merge_keys(best, sort_keys(c, 32, lane), lane);
        }
        bar = key_value(__shfl_sync(kFull, best, beams - 1));
        hits = list_hits(scan, hit, spans, bar, lane);
        best = 0;
    }
    Key last = bar > -INFINITY ? (Key)ordered(bar + 0.0f) << 32 : 0;  // candidates are larger
    const int total = hits * per * kSelUnroll;  // groups of N to look at, two in flight a lane
    const float inv_per = 1.0f / (float)per;
#pragma unroll 1
    for (int j0 = 0; j0 < total; j0 += 64) {
        float x[2][N];
        int at[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = j0 + u * 32 + lane, pb = j / kSelUnroll;
            at[u] = c1;
            if (j < total) {
                const int q = (int)(((float)pb + 0.5f) * inv_per);  // pb / per
                const int h = hit[q], batch = (h >> 5) * per + pb - q * per;
                const int in = (j % kSelUnroll * 32 + (h & 31)) * N, c = c0 + batch * kBatch + in;
                at[u] = c;
                const T *src = kept ? reinterpret_cast<const T *>(scan.ring[batch % kStages] + skew) + in : row + c;
                if (skew == 0 && c + N <= c1) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(src);
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < N; ++e) x[u][e] = element<T>(ws[e * (int)sizeof(T) / 4], e & 1);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) x[u][e] = c + e < c1 ? to_f32(src[e]) : -INFINITY;
                }
            }
        }
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float v = u ? x[1][e] : x[0][e];
                const int i = (u ? at[1] : at[0]) + e;
                const bool in = i < c1 && v >= bar;  // (NaN is not)
                if (!__any_sync(kFull, in)) continue;
                const Key c = in ? make_key(v, i) : 0;
                append(cand, c, c > last, count, lane);
                if (count >= 32) {
                    best = take_32(cand, best, count, lane);
                    const Key kth = __shfl_sync(kFull, best, beams - 1);
                    last = kth > last ? kth : last;
                }
            }
        }
    }
    if (count > 0) best = take_32(cand, best, count, lane);
    __syncwarp();  // the next scan of this warp writes here again
    const float top = warp_max(m);
    // an infinite top: lanes that saw it have counted it, the others add nothing
    if (m != top) sum = m > -INFINITY ? sum * (double)exp2_approx((m - top) * kLog2e) : 0.0;
    sum = warp_sum(sum);
    if (lane < beams) out.best[lane] = best;
    if (lane == 0) {
        out.top = top;
        out.sum = sum;
    }
}

// What a line's merge works on in shared memory.
struct Merge {
    double score[TRBA_MAX_BEAMS][TRBA_MAX_BEAMS];
    int tok[TRBA_MAX_BEAMS][TRBA_MAX_BEAMS];
    Key cand[16][kBuffer];  // a warp's each
};

// Joins what was found in the rows' segments and picks the line's best: a warp
// a beam joins the segments of its row, then the first warp merges the beams'
// lists, its lane b at the head of beam b's.  find(b, s): segment s of beam b.
template <class F>
__device__ __forceinline__ void merge_line(F find, int segs, float my_score, unsigned alive, unsigned over, int beams,
                                           int eos, i64 slot0, Merge &mg, float *out_scores, int32_t *out_tokens,
                                           int32_t *out_parents, uint8_t *out_finished) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll 1
    for (int b = warp; b < beams; b += warps) {
        const float sc = __shfl_sync(kFull, my_score, b);
        double out = -INFINITY;
        int tok = kNone;
        if ((alive >> b & 1) && (over >> b & 1)) {
            if (lane == 0) {
                out = (double)sc;
                tok = eos;
            }
        } else if (alive >> b & 1) {
            // the row's sum; and a bar: the row's beams-th best is at least any segment's
            float top = -INFINITY;
            double sum = 0.0;
            unsigned bar = 0;
#pragma unroll 1
            for (int s = lane; s < segs; s += 32) {
                const Found *f = find(b, s);
                const float m = f->top;
                const double part = f->sum;
                bar = max(bar, (unsigned)(f->best[beams - 1] >> 32));
                if (m > top) {
                    sum *= (double)exp2_approx((top - m) * kLog2e);
                    top = m;
                }
                if (m > -INFINITY) sum += m == top ? part : part * (double)exp2_approx((m - top) * kLog2e);
            }
            bar = __reduce_max_sync(kFull, bar);
            const float all = warp_max(top);
            if (top != all) sum = top > -INFINITY ? sum * (double)exp2_approx((top - all) * kLog2e) : 0.0;
            const double lse = log(warp_sum(sum));
            Key best = segs == 1 && lane < beams ? find(b, 0)->best[lane] : 0;
            if (segs > 1) {
                Key *cand = mg.cand[warp];
                int count = 0;
                const float inv = 1.0f / (float)beams;
#pragma unroll 1
                for (int e0 = 0; e0 < segs * beams; e0 += 128) {
                    Key key[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int e = e0 + u * 32 + lane, s = (int)(((float)e + 0.5f) * inv);  // e / beams
                        key[u] = e < segs * beams ? find(b, s)->best[e - s * beams] : 0;
                    }
#pragma unroll 1
                    for (int u = 0; u < 4; ++u) {
                        const Key c = u == 0 ? key[0] : u == 1 ? key[1] : u == 2 ? key[2] : key[3];
                        append(cand, c, c != 0 && (unsigned)(c >> 32) >= bar, count, lane);
                        if (count >= 32) best = take_32(cand, best, count, lane);
                    }
                }
                if (count > 0) best = take_32(cand, best, count, lane);
                __syncwarp();
            }
            if (lane < beams && best) {
                const float x = key_value(best);
                out = (double)sc + ((x == all ? 0.0 : (double)x - (double)all) - lse);
                tok = key_index(best);
            }
        }
        if (!((float)out > -INFINITY)) out = -INFINITY;
        if (lane < beams) {
            mg.score[b][lane] = out + 0.0;  // no -0: scores are compared by their bits below
            mg.tok[b][lane] = tok;
        }
    }
    __syncthreads();
    if (warp != 0) return;
    int head = 1;
    double v = lane < beams ? mg.score[lane][0] : -INFINITY;
    double v1 = lane < beams && beams > 1 ? mg.score[lane][1] : -INFINITY;  // the next, ahead of its use
    unsigned key = ordered((float)v);
#pragma unroll 1
    for (int k = 0; k < beams; ++k) {
        // the largest in f32 (rounding keeps the order); only lanes that tie there compare in f64
        const unsigned most = __reduce_max_sync(kFull, key);
        unsigned tied = __ballot_sync(kFull, key == most);
        int who = __ffs(tied) - 1;
        const bool none = most == ordered(-INFINITY);
        if ((tied & (tied - 1)) && !none) {
            double top = __shfl_sync(kFull, v, who);
#pragma unroll 1
            while (tied &= tied - 1) {  // ties between beams go to the lower beam
                const int w = __ffs(tied) - 1;
                const double o = __shfl_sync(kFull, v, w);
                if (o > top) {
                    top = o;
                    who = w;
                }
            }
        }
        if (lane == who) {
            const int tok = none ? max(eos, 0) : mg.tok[lane][head - 1];
            out_scores[slot0 + k] = (float)v;
            out_tokens[slot0 + k] = tok;
            out_parents[slot0 + k] = none ? k : lane;
            out_finished[slot0 + k] = eos >= 0 && (none || tok == eos || (over >> lane & 1));
            ++head;
            v = v1;
            key = ordered((float)v);
            v1 = head < beams && lane < beams ? mg.score[lane][head] : -INFINITY;
        }
    }
}

// A line's beams: bit b of `alive` when beam b has a score above -inf (a NaN
// has not), of `over` when it is finished.
struct Line {
    float score;  // lane b: beam b's
    unsigned alive, over;
    __device__ __forceinline__ void load(const float *scores, const uint8_t *finished, i64 slot0, int beams) {
        const int lane = threadIdx.x & 31;
        score = lane < beams ? scores[slot0 + lane] : -INFINITY;
        const bool fin = lane < beams && finished && finished[slot0 + lane];
        alive = __ballot_sync(kFull, score > -INFINITY);
        over = __ballot_sync(kFull, fin);
    }
};

// Short rows: a CTA a line, a warp a row.  Bound by latency: a read of the row,
// its sort, the logarithm and `beams` rounds of picking, one after the other
// (one line of 5 beams over 130 f32: 6.4 us; 512 lines of 5: 8.4; a
// launch of nothing takes about 2).  One kernel, because a second launch would
// add half as much again.
template <class T>
__global__ void __launch_bounds__(512) select_line_kernel(const T *__restrict__ logits, i64 ld, const float *scores,
                                                          const uint8_t *finished, int beams, int vocab, int eos,
                                                          float *out_scores, int32_t *__restrict__ out_tokens,
                                                          int32_t *__restrict__ out_parents, uint8_t *out_finished) {
    extern __shared__ __align__(16) uint8_t sel_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const i64 slot0 = (i64)blockIdx.x * beams;
    Merge &mg = *reinterpret_cast<Merge *>(sel_smem);
    Scan *scan = reinterpret_cast<Scan *>(&mg + 1);
    Found *found = reinterpret_cast<Found *>(scan + warps);
    Line line;
    line.load(scores, finished, slot0, beams);
#pragma unroll 1
    for (int b = warp; b < beams; b += warps)
        if ((line.alive & ~line.over) >> b & 1)
            scan_segment<T>(logits + (slot0 + b) * ld, 0, vocab, beams, lane, scan[warp], found[b]);
    __syncwarp();  // (the warp that scanned a row joins it too)
    merge_line([&](int b, int) -> const Found * { return found + b; }, 1, line.score, line.alive, line.over, beams, eos,
               slot0, mg, out_scores, out_tokens, out_parents, out_finished);
}

// Long rows, first part: a warp a segment of a row, to the workspace.  Warps
// of dead and finished beams end at once; the others come and go, so that
// some read while others pick their best.  64 lines of 10 beams over 65536 f32
// (134 MB of live rows): 36 us with the merge, 3.7 TB/s of 6.5; what bounds it
// is the instructions an element takes (a conversion, a maximum, a subtraction
// and product, an exponential and an addition; issue slots 47% used with 22
// warps a SM) and the second look's latency, not the bytes.  Seven CTAs a SM of
// 64 registers a thread are what keeps enough reads in flight.
constexpr int kScanWarps = 4;
template <class T>
__global__ void __launch_bounds__(kScanWarps * 32, 7) select_scan_kernel(
    const T *__restrict__ logits, i64 ld, const float *__restrict__ scores, const uint8_t *__restrict__ finished,
    int beams, int vocab, int segs, int seg_len, i64 units, Found *__restrict__ found) {
    __shared__ Scan scan[kScanWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const i64 u = (i64)blockIdx.x * kScanWarps + warp;
    if (u >= units) return;
    const i64 row = u / segs;
    if (!(scores[row] > -INFINITY) || (finished && finished[row])) return;
    const int c0 = (int)(u - row * segs) * seg_len;
    scan_segment<T>(logits + row * ld, c0, min(vocab, c0 + seg_len), beams, lane, scan[warp], found[u]);
}

// Second part: a CTA a line; bound by latency, as the short rows are (6 to 9
// us for 64 lines of 10 beams, 16 segments each).
__global__ void __launch_bounds__(512) select_merge_kernel(const Found *__restrict__ found, int segs,
                                                           const float *scores, const uint8_t *finished, int beams,
                                                           int eos, float *out_scores, int32_t *__restrict__ out_tokens,
                                                           int32_t *__restrict__ out_parents, uint8_t *out_finished) {
    extern __shared__ __align__(16) uint8_t sel_smem[];
    const i64 slot0 = (i64)blockIdx.x * beams;
    Line line;
    line.load(scores, finished, slot0, beams);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the first part ends
    merge_line([&](int b, int s) -> const Found * { return found + (slot0 + b) * segs + s; }, segs, line.score,
               line.alive, line.over, beams, eos, slot0, *reinterpret_cast<Merge *>(sel_smem), out_scores, out_tokens,
               out_parents, out_finished);
}

// -------------------------------------------------------------- reordering --
// A copy, bound by memory.  A warp moves a piece of a row at a time, 4 units of
// 16 bytes or 8 smaller ones a lane in flight.  Rows whose addresses are all
// multiples of 4, 8 or 16 bytes go in such units; others in 4-byte words of the
// destination, each put together from the two source words it lies in.  (Wider
// units, put together from aligned ones as the selection's scan does, were not
// tried.)
constexpr int kMaxStates = 16;
__host__ __device__ constexpr int moves_of(int vec) { return vec == 16 ? 4 : 8; }
struct StateView {
    const char *src;
    char *dst;
    i64 bytes, src_row, dst_row, src_mid, dst_mid, src_outer, dst_outer;
    int mid, per_row;  // parts of a row; pieces of a part
    int vec;           // unit in bytes, 0: words that are put together
    int first;         // the state's first piece in the launch
};
struct StateViews {
    StateView s[kMaxStates];
    int n, pieces;
};

template <class V, bool STREAM>
__device__ __forceinline__ void move_units(const char *src, char *dst, int units, int lane) {
    constexpr int kMoves = moves_of(sizeof(V));
    const V *from = reinterpret_cast<const V *>(src) + lane;
    V *to = reinterpret_cast<V *>(dst) + lane;
    V v[kMoves];
    if (units >= kMoves * 32) {
#pragma unroll
        for (int u = 0; u < kMoves; ++u) v[u] = STREAM ? __ldcs(from + u * 32) : from[u * 32];
#pragma unroll
        for (int u = 0; u < kMoves; ++u) {
            if (STREAM) __stcs(to + u * 32, v[u]);
            else to[u * 32] = v[u];
        }
    } else {
        units -= lane;
#pragma unroll
        for (int u = 0; u < kMoves; ++u)
            if (u * 32 < units) v[u] = from[u * 32];
#pragma unroll
        for (int u = 0; u < kMoves; ++u)
            if (u * 32 < units) to[u * 32] = v[u];
    }
}

// `bytes` from any src to any dst, at most moves_of(0) * 128.
__device__ __noinline__ void move_bytes(const char *src, char *dst, int bytes, int lane) {
    const int head = min(bytes, (int)(-reinterpret_cast<uintptr_t>(dst) & 3)), words = (bytes - head) >> 2;
    if (lane < head) dst[lane] = src[lane];
    const uintptr_t at = reinterpret_cast<uintptr_t>(src + head);
    const uint32_t *w = reinterpret_cast<const uint32_t *>(at & ~(uintptr_t)3);
    const int shift = (int)(at & 3) * 8;
    constexpr int kMoves = moves_of(0);
    uint32_t lo[kMoves], hi[kMoves];
#pragma unroll
    for (int u = 0; u < kMoves; ++u) {
        const int i = u * 32 + lane;
        if (i < words) {
            lo[u] = w[i];
            hi[u] = shift ? w[i + 1] : 0;  // holds bytes of this word
        }
    }
#pragma unroll
    for (int u = 0; u < kMoves; ++u) {
        const int i = u * 32 + lane;
        if (i < words) reinterpret_cast<uint32_t *>(dst + head)[i] = __funnelshift_r(lo[u], hi[u], shift);
    }
    const int done = head + words * 4;
    if (lane < bytes - done) dst[done + lane] = src[done + lane];
}

// 4 layer states of 5 MB: 10.9 us (3.8 TB/s read and written, the L2 cache
// serving part); 8 cache tensors of 87 MB: 198 us (7.0 TB/s counting every row
// as read, parents that repeat being read once from memory), which is what a
// plain copy of as many bytes takes.
// STREAM: more than stays in the L2 cache is moved, past it (203 us instead of
// 214 for 0.7 GB, both with 8 CTAs a SM).
template <bool STREAM>
__global__ void __launch_bounds__(256, 4) beam_reorder_kernel(const __grid_constant__ StateViews st,
                                                           const int32_t *__restrict__ parents, int rows, int beams) {
    const int lane = threadIdx.x & 31, warps = gridDim.x * 8;
    int k = 0;
    for (int piece = blockIdx.x * 8 + (threadIdx.x >> 5); piece < st.pieces; piece += warps) {
        while (k + 1 < st.n && piece >= st.s[k + 1].first) ++k;
        const StateView &s = st.s[k];
        const int local = piece - s.first, part = s.per_row == 1 ? local : local / s.per_row;
        const int q = local - part * s.per_row, row_o = s.mid == 1 ? part : part / s.mid, mid = part - row_o * s.mid;
        const int outer = row_o < rows ? 0 : row_o / rows, row = row_o - outer * rows;
        const int p = parents[row];
        if ((unsigned)p >= (unsigned)beams) continue;
        const int from = row - row % beams + p;
        const int unit = s.vec ? s.vec : 4;
        const i64 at = (i64)q * (moves_of(s.vec) * 32) * unit;
        const int left = (int)min(s.bytes - at, (i64)moves_of(s.vec) * 32 * unit);
        const char *src = s.src + outer * s.src_outer + (i64)from * s.src_row + mid * s.src_mid + at;
        char *dst = s.dst + outer * s.dst_outer + (i64)row * s.dst_row + mid * s.dst_mid + at;
        if (s.vec == 16) move_units<uint4, STREAM>(src, dst, left / 16, lane);
        else if (s.vec == 8) move_units<uint2, STREAM>(src, dst, left / 8, lane);
        else if (s.vec == 4) move_units<uint32_t, STREAM>(src, dst, left / 4, lane);
        else move_bytes(src, dst, left, lane);
    }
}

// --------------------------------------------------------------- sequences --
// A path is a chain of dependent reads, so the walk goes over shared memory
// and in parallel: the steps are cut into segments, one thread a segment and
// slot finds where the slot leads to at the segment's start, the segments'
// maps are composed, and a second walk from the right slots notes the path.
// A CTA takes `group` lines, or a part of one line's beams (all CTAs of a line
// read its parents).  Steps that do not fit go in chunks, last first.
// 512 lines of 5 beams, 21 steps 6.4 us, most of it launch and latency.  16 lines
// of 16 beams, 2000 steps 16.5 us (0.36 TB/s), where a thread a path over device
// memory took 1007: with a line's beams shared by 1 / 2 / 4 / 8 CTAs it takes
// 30.8 / 22.6 / 18.5 / 16.5 us, so about 2 us of the second walk and the writing
// are left, and 14 that sharing by beams does not divide: the launch, reading
// all parents of the line, the first walk (63 dependent reads) and the
// composition (32), in every CTA.
constexpr uint8_t kLost = 255;  // behind a parent out of range

constexpr int kTraceSmem = 96 * 1024;

struct Trace {
    const int32_t *tokens, *parents;
    int32_t *seq, *lengths;
    int steps, lines, beams, eos, pad;
    int group, segs, chunk, splits;
    bool fours;  // parents can be read four at a time
};

constexpr int kTraceLoads = 4;  // loads in flight a thread

// A thread's walk over [major][minor] in strides, without a division a step.
struct Index {
    int major, minor, minors, up, right;
    __device__ __forceinline__ Index(int first, int minors_, int stride)
        : major(first / minors_), minor(first % minors_), minors(minors_), up(stride / minors_), right(stride % minors_) {}
    __device__ __forceinline__ void next() {
        major += up;
        minor += right;
        if (minor >= minors) {
            minor -= minors;
            ++major;
        }
    }
};
// The first slot of a slot's line.
__device__ __forceinline__ int line_of(int k, int beams) { return k - k % beams; }

__global__ void __launch_bounds__(1024) beam_sequences_kernel(const Trace a) {
    extern __shared__ __align__(16) uint8_t tr_smem[];
    const int threads = blockDim.x;
    const int gk = a.group * a.beams;  // slots of the CTA's lines
    uint8_t *par = tr_smem;            // [chunk][gk]
    uint8_t *path = par + a.chunk * gk;
    uint8_t *map = path + a.chunk * gk;  // [segs][gk], then the segments' entry slots
    uint8_t *end = map + a.segs * gk;    // [gk]: where the paths stand
    int *len = reinterpret_cast<int *>(tr_smem + ((2 * a.chunk * gk + (a.segs + 1) * gk + 3) & ~3));
    const int line0 = blockIdx.x * a.group, slots = min(a.group, a.lines - line0) * a.beams;
    // the slots whose sequences this CTA writes
    const int k0 = slots * blockIdx.y / a.splits, own = slots * (blockIdx.y + 1) / a.splits - k0;
    const i64 n = (i64)a.lines * a.beams, base = (i64)line0 * a.beams;
    const int32_t *__restrict__ parents = a.parents + base, *__restrict__ tokens = a.tokens + base;
    for (int e = threadIdx.x; e < slots; e += threads) {
        end[e] = (uint8_t)(e % a.beams);
        len[e] = a.steps;
    }
    for (int hi = a.steps; hi > 0; hi -= a.chunk) {  // the steps [lo, hi)
        const int lo = max(0, hi - a.chunk), c = hi - lo;
        __syncthreads();
        // (unsigned: what is out of range, below 0 too, is no slot)
        const auto slot_of = [&](int p) { return (unsigned)p < (unsigned)a.beams ? (unsigned)p : (unsigned)kLost; };
        const int32_t *row = parents + lo * n;
        if (a.fours) {  // four slots at a time
            Index at(threadIdx.x, slots >> 2, threads);  // step, slot / 4
            for (int e0 = threadIdx.x; e0 < c * (slots >> 2); e0 += threads * 4) {
                int4 p[4];
                int to[4];
#pragma unroll
                for (int u = 0; u < 4; ++u, at.next()) {
                    to[u] = at.major < c ? at.major * gk + at.minor * 4 : -1;
                    p[u] = make_int4(0, 0, 0, 0);  // step 0 has no parents
                    if (to[u] >= 0 && lo + at.major) p[u] = *reinterpret_cast<const int4 *>(row + at.major * n + at.minor * 4);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (to[u] >= 0)
                        *reinterpret_cast<unsigned *>(par + to[u]) = slot_of(p[u].x) | slot_of(p[u].y) << 8 |
                                                                     slot_of(p[u].z) << 16 | slot_of(p[u].w) << 24;
            }
        } else {
            Index at(threadIdx.x, slots, threads);  // step, slot
            for (int e0 = threadIdx.x; e0 < c * slots; e0 += threads * kTraceLoads) {
                int p[kTraceLoads], to[kTraceLoads];
#pragma unroll
                for (int u = 0; u < kTraceLoads; ++u, at.next()) {
                    to[u] = at.major < c ? at.major * gk + at.minor : -1;
                    p[u] = to[u] >= 0 && lo + at.major ? row[at.major * n + at.minor] : 0;
                }
#pragma unroll
                for (int u = 0; u < kTraceLoads; ++u)
                    if (to[u] >= 0) par[to[u]] = (uint8_t)slot_of(p[u]);
            }
        }
        __syncthreads();
        const int per = (c + a.segs - 1) / a.segs;
        for (int w = threadIdx.x; w < a.segs * slots; w += threads) {
            const int s = w / slots, e = w - s * slots, l = e - e % a.beams;
            uint8_t x = (uint8_t)(e % a.beams);
            for (int t = min(c, (s + 1) * per) - 1; t >= s * per && x != kLost; --t) x = par[t * gk + l + x];
            map[s * gk + e] = x;
        }
        __syncthreads();
        // maps become entry slots; a segment's map is read by all slots of its
        // line, so the entries wait in the path's first rows
        for (int e = threadIdx.x; e < slots; e += threads) {
            const int l = e - e % a.beams;
            uint8_t x = end[e];
            for (int s = a.segs - 1; s >= 0; --s) {
                path[s * gk + e] = x;
                if (x != kLost) x = map[s * gk + l + x];
            }
            end[e] = x;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.segs * gk; e += threads) map[e] = path[e];
        __syncthreads();
        for (int w = threadIdx.x; w < a.segs * own; w += threads) {
            const int s = w / own, e = k0 + w - s * own, l = e - e % a.beams;
            uint8_t x = map[s * gk + e];
            for (int t = min(c, (s + 1) * per) - 1; t >= s * per; --t) {
                path[t * gk + e] = x;
                if (x != kLost) x = par[t * gk + l + x];
            }
        }
        __syncthreads();
        Index it(threadIdx.x, c, threads);  // slot, step
        for (int e0 = threadIdx.x; e0 < c * own; e0 += threads * kTraceLoads) {
            int tok[kTraceLoads], k[kTraceLoads], t[kTraceLoads], x[kTraceLoads];
#pragma unroll
            for (int u = 0; u < kTraceLoads; ++u, it.next()) {
                k[u] = it.major < own ? k0 + it.major : -1, t[u] = it.minor;
                x[u] = k[u] >= 0 ? path[t[u] * gk + k[u]] : kLost;
                tok[u] = x[u] == kLost ? a.pad : tokens[(lo + t[u]) * n + line_of(k[u], a.beams) + x[u]];
            }
#pragma unroll
            for (int u = 0; u < kTraceLoads; ++u) {
                if (k[u] < 0) break;
                if (x[u] == kLost) atomicMin(&len[k[u]], -1);
                else if (tok[u] == a.eos) atomicMin(&len[k[u]], lo + t[u]);
                a.seq[(base + k[u]) * a.steps + lo + t[u]] = tok[u];
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < own; e += threads) a.lengths[base + k0 + e] = len[k0 + e];
    for (int e = threadIdx.x >> 5; e < own; e += threads / 32)  // what follows the end
        for (int t = max(0, len[k0 + e]) + (threadIdx.x & 31); t < a.steps; t += 32)
            a.seq[(base + k0 + e) * a.steps + t] = a.pad;
}

int launched() {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
    return (int)e;
}

// How a selection runs: rows of up to two batches whole (segs = 0), longer
// ones in segments of whole batches: one round of warps on the device, but no
// segment so short that picking its best (and joining them, with many beams)
// costs more than reading it, and up to 128 segments (1 Mi f32 tokens) none of
// more batches than there are spans to remember, so that a second look is at
// one batch's groups.  With 2 / 4 / 8 /
// 16 / 24 / 32 batches a segment, 64 lines of 10 beams, 65536 f32 take 68 / 50 /
// 41 / 36 / 39 / 41 us, 16 lines of 32 beams, 20000 bf16 51 / 39 / 35 / 35 / 37 /
// 37, one line of 5 beams, 32000 bf16 11 / 12 / 15 / 19 / 19 / 27.
struct Plan {
    int segs, len;
    Plan(int lines, int beams, int vocab, int size) {
        const int batch = kSelUnroll * 32 * 16 / size, batches = (vocab - 1) / batch + 1;
        segs = len = 0;
        if (batches <= 2) return;
        const i64 all = (i64)lines * beams * batches, slots = (i64)sm_count() * 7 * kScanWarps;
        const int least = beams > 8 ? beams / 4 : 2, most = 16;
        int per = all >= slots * most ? most : (int)(all / slots) + 1;
        if (per < least) per = least;
        if (per < (batches + 127) / 128) per = (batches + 127) / 128;
        segs = (batches + per - 1) / per;
        len = (batches + segs - 1) / segs * batch;
        segs = (vocab - 1) / len + 1;
    }
};

int size_of(int dtype) { return dtype == TRBA_F32 ? 4 : 2; }

// Raises a kernel's shared-memory limit, once a device.
template <class K>
int allow_smem(K kernel, std::atomic<unsigned long long> &done) {
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) {
        report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
        return (int)e;
    }
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

// The widest unit that every address of a state is a multiple of (0: none).
int unit_of(const trba_beam_state &s) {
    i64 bits = (i64)reinterpret_cast<uintptr_t>(s.src) | (i64)reinterpret_cast<uintptr_t>(s.dst) | s.bytes | s.src_row |
               s.dst_row;
    if (s.mid > 1) bits |= s.src_mid | s.dst_mid;
    if (s.outer > 1) bits |= s.src_outer | s.dst_outer;
    return !(bits & 15) ? 16 : !(bits & 7) ? 8 : !(bits & 3) ? 4 : 0;
}
// Pieces of a part of a row of a state, and the most that a launch counts: a
// warp's next piece is still below 2^31.
i64 pieces_of(const trba_beam_state &s, int vec) { return (s.bytes - 1) / (moves_of(vec) * 32 * (vec ? vec : 4)) + 1; }
constexpr i64 kMostPieces = 2147483647ll - (1 << 20);

template <class T>
int select(const void *logits, i64 ld, const float *scores, const uint8_t *finished, int lines, int beams, int vocab,
           int eos, float *out_scores, int32_t *out_tokens, int32_t *out_parents, uint8_t *out_finished,
           void *workspace, cudaStream_t st) {
    const Plan plan(lines, beams, vocab, (int)sizeof(T));
    if (plan.segs == 0) {
        static std::atomic<unsigned long long> sized{0};
        if (const int e = allow_smem(select_line_kernel<T>, sized)) return e;
        // More lines than SMs: 8 warps, so that several CTAs fit on a SM and one
        // picks while others read (512 lines of 32 beams, 130 f32: 72 us with 8
        // warps, 82 with 16; of 16 beams, 200 f16: 31 and 37); few lines are
        // quickest with a warp for every row.
        const int most = lines > sm_count() ? 8 : 16, warps = beams < most ? beams : most;
        const size_t smem = sizeof(Merge) + sizeof(Scan) * warps + sizeof(Found) * beams;
        select_line_kernel<T><<<lines, warps * 32, smem, st>>>(static_cast<const T *>(logits), ld, scores, finished,
                                                               beams, vocab, eos, out_scores, out_tokens, out_parents,
                                                               out_finished);
        return launched();
    }
    static std::atomic<unsigned long long> sized{0};
    const int warps = beams < 16 ? beams : 16;
    Found *found = static_cast<Found *>(workspace);
    const i64 units = (i64)lines * beams * plan.segs;
    select_scan_kernel<T><<<(unsigned)((units + kScanWarps - 1) / kScanWarps), kScanWarps * 32, 0, st>>>(
        static_cast<const T *>(logits), ld, scores, finished, beams, vocab, plan.segs, plan.len, units, found);
    if (const int e = launched()) return e;
    if (const int e = allow_smem(select_merge_kernel, sized)) return e;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(lines);
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = sizeof(Merge);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, select_merge_kernel, static_cast<const Found *>(found), plan.segs, scores, finished, beams,
                       eos, out_scores, out_tokens, out_parents, out_finished);
    return launched();
}

}  // namespace
}  // namespace trba

using namespace trba;

extern "C" {

long long trba_beam_select_workspace(int dtype, int lines, int beams, int vocab) {
    if (lines <= 0 || beams <= 0 || beams > TRBA_MAX_BEAMS || vocab <= 0 || vocab > (1 << 30) ||
        (dtype != TRBA_F32 && dtype != TRBA_BF16 && dtype != TRBA_F16))
        return 0;
    return (long long)sizeof(Found) * lines * beams * Plan(lines, beams, vocab, size_of(dtype)).segs;
}

int trba_beam_select(const void *logits, int dtype, long long ld, const float *scores, const uint8_t *finished,
                     int lines, int beams, int vocab, int eos, float *out_scores, int32_t *out_tokens,
                     int32_t *out_parents, uint8_t *out_finished, void *workspace, long long workspace_bytes,
                     void *stream) {
    TRBA_REQUIRE_RET(lines >= 0 && beams > 0 && beams <= TRBA_MAX_BEAMS && vocab > 0 && vocab <= (1 << 30) &&
                         ld >= vocab && (i64)beams * vocab < (1ll << 31) && (i64)lines * beams < (1ll << 24),
                     "trba_beam_select: bad sizes", -1);
    TRBA_REQUIRE_RET(eos >= -1 && eos < vocab && (eos >= 0 || !finished),
                     "trba_beam_select: eos outside the vocabulary, or finished beams without an end token", -1);
    TRBA_REQUIRE_RET(dtype == TRBA_F32 || dtype == TRBA_BF16 || dtype == TRBA_F16,
                     "trba_beam_select: unknown element type", -1);
    if (lines == 0) return 0;
    TRBA_REQUIRE_RET(logits && scores && out_scores && out_tokens && out_parents && out_finished,
                     "trba_beam_select: null pointer", -1);
    TRBA_REQUIRE_RET(reinterpret_cast<uintptr_t>(logits) % size_of(dtype) == 0,
                     "trba_beam_select: logits are not aligned to their elements", -1);
    const long long need = trba_beam_select_workspace(dtype, lines, beams, vocab);
    TRBA_REQUIRE_RET(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                     "trba_beam_select: workspace missing, too small or not aligned to 16 bytes", -1);
    cudaStream_t st = as_stream(stream);
    if (dtype == TRBA_F32)
        return select<float>(logits, ld, scores, finished, lines, beams, vocab, eos, out_scores, out_tokens,
                             out_parents, out_finished, workspace, st);
    if (dtype == TRBA_BF16)
        return select<__nv_bfloat16>(logits, ld, scores, finished, lines, beams, vocab, eos, out_scores, out_tokens,
                                     out_parents, out_finished, workspace, st);
    return select<__half>(logits, ld, scores, finished, lines, beams, vocab, eos, out_scores, out_tokens, out_parents,
                          out_finished, workspace, st);
}

int trba_beam_reorder(const trba_beam_state *states, int n_states, const int32_t *parents, int lines, int beams,
                      void *stream) {
    TRBA_REQUIRE_RET(n_states >= 0 && lines >= 0 && beams > 0 && beams <= TRBA_MAX_BEAMS,
                     "trba_beam_reorder: bad sizes", -1);
    if (n_states == 0 || lines == 0) return 0;
    TRBA_REQUIRE_RET(states && parents, "trba_beam_reorder: null pointer", -1);
    const i64 rows = (i64)lines * beams;
    TRBA_REQUIRE_RET(rows < (1ll << 24), "trba_beam_reorder: bad sizes", -1);
    for (int i = 0; i < n_states; ++i) {
        const trba_beam_state &s = states[i];
        TRBA_REQUIRE_RET(s.bytes >= 0 && s.mid >= 0 && s.outer >= 0, "trba_beam_reorder: negative size", -1);
        TRBA_REQUIRE_RET((s.src && s.dst) || s.bytes == 0 || s.mid == 0 || s.outer == 0,
                         "trba_beam_reorder: null state", -1);
        TRBA_REQUIRE_RET(s.mid < (1ll << 31) && s.outer < (1ll << 31), "trba_beam_reorder: bad sizes", -1);
        if (s.bytes == 0 || s.mid == 0 || s.outer == 0) continue;
        const double all = (double)pieces_of(s, unit_of(s)) * (double)s.mid * (double)s.outer * (double)rows;
        TRBA_REQUIRE_RET(all <= (double)kMostPieces, "trba_beam_reorder: a state is too large for one launch", -1);
    }
    int i = 0;
    while (i < n_states) {
        StateViews v{};
        i64 pieces = 0, bytes = 0;
        for (; i < n_states && v.n < kMaxStates; ++i) {
            const trba_beam_state &s = states[i];
            if (s.bytes == 0 || s.mid == 0 || s.outer == 0) continue;
            StateView &d = v.s[v.n];
            d.vec = unit_of(s);
            const i64 per_row = pieces_of(s, d.vec), mine = per_row * s.mid * s.outer * rows;
            if (pieces + mine > kMostPieces) break;  // the next launch takes it
            d.first = (int)pieces;
            pieces += mine;
            bytes += s.bytes * s.mid * s.outer * rows;
            d.src = static_cast<const char *>(s.src);
            d.dst = static_cast<char *>(s.dst);
            d.bytes = s.bytes, d.per_row = (int)per_row, d.mid = (int)s.mid;
            d.src_row = s.src_row, d.dst_row = s.dst_row;
            d.src_mid = s.src_mid, d.dst_mid = s.dst_mid;
            d.src_outer = s.src_outer, d.dst_outer = s.dst_outer;
            ++v.n;
        }
        if (v.n == 0) break;  // only empty states were left
        v.pieces = (int)pieces;
        // Rounds of CTAs even out the SMs' shares: 0.7 GB moved by 3 / 8 / 64
        // CTAs a SM takes 213 / 219 / 195 us, 21 MB 10.8 us up to 32 and 14 at 64.
        const bool past = bytes > (64ll << 20);
        const i64 want = (pieces + 7) / 8, cap = (i64)sm_count() * (past ? 64 : 16);
        const int grid = (int)(want < cap ? want : cap);
        if (past)
            beam_reorder_kernel<true><<<grid, 256, 0, as_stream(stream)>>>(v, parents, (int)rows, beams);
        else
            beam_reorder_kernel<false><<<grid, 256, 0, as_stream(stream)>>>(v, parents, (int)rows, beams);
        if (const int e = launched()) return e;
    }
    return 0;
}

int trba_beam_sequences(const int32_t *tokens, const int32_t *parents, int steps, int lines, int beams, int eos,
                        int pad, int32_t *sequences, int32_t *lengths, void *stream) {
    TRBA_REQUIRE_RET(steps >= 0 && lines >= 0 && beams > 0 && beams <= TRBA_MAX_BEAMS &&
                         (i64)lines * beams < (1ll << 24) && steps < (1 << 24),
                     "trba_beam_sequences: bad sizes", -1);
    if (lines == 0) return 0;
    TRBA_REQUIRE_RET(lengths && (steps == 0 || (tokens && parents && sequences)), "trba_beam_sequences: null pointer",
                     -1);
    Trace a{};
    a.tokens = tokens, a.parents = parents, a.seq = sequences, a.lengths = lengths;
    a.steps = steps, a.lines = lines, a.beams = beams, a.eos = eos, a.pad = pad;
    // About as many segments as steps in a segment, and lines until a CTA's
    // threads have a walk each, as long as that leaves a CTA for every SM;
    // few lines of many steps are split by their beams instead.
    a.segs = 1;
    while (a.segs < 64 && a.segs * a.segs * 2 < steps) a.segs *= 2;
    const int threads = steps < 128 ? 256 : 1024;
    a.group = threads / (beams * a.segs);
    const int even = (lines + sm_count() - 1) / sm_count();
    if (a.group > even) a.group = even;
    if (a.group < 1) a.group = 1;
    a.splits = 1;
    while (steps >= 128 && a.group == 1 && a.splits < 8 && 2 * a.splits <= beams && 2 * a.splits * lines <= sm_count())
        a.splits *= 2;
    const int gk = a.group * beams;
    a.fours = beams % 4 == 0 && reinterpret_cast<uintptr_t>(parents) % 16 == 0;
    a.chunk = kTraceSmem / (2 * gk);
    if (a.chunk > steps) a.chunk = steps;
    if (a.chunk < a.segs) a.chunk = a.segs;  // (the entry slots pass through the path's rows)
    const size_t smem = (((size_t)2 * a.chunk * gk + (size_t)(a.segs + 1) * gk + 3) & ~(size_t)3) + (size_t)gk * 4;
    static std::atomic<unsigned long long> sized{0};
    if (const int e = allow_smem(beam_sequences_kernel, sized)) return e;
    beam_sequences_kernel<<<dim3((lines + a.group - 1) / a.group, a.splits), threads, smem, as_stream(stream)>>>(a);
    return launched();
}

}  // extern "C"
