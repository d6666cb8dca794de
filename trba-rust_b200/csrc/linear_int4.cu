// Linear layer with 4-bit weights and group scales for the few rows of a
// decoding step (include/trba_ops.h, LinearInt4).  No counterpart in the
// reference; the quantisation rule is LinearInt8's (src/linear.rs:53-59) for
// 4 bits and groups.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdlib>
#include <new>

#include "common.cuh"
#include "trba_decode.h"
#include "trba_ops.h"

// Weight layout, made once when a layer is created: outputs in tiles of 16,
// inputs in chunks of 128, so that a warp streams one tile's chunks as
// consecutive 1 KB blocks with fully coalesced 16-byte loads that are already
// the A fragments of mma.m16n8k16.  In a block, lane l = 4 g + t has 16 bytes
// of row g (first 512 bytes) and 16 of row g + 8; their word w holds the
// codes of inputs 32 w + 8 t .. + 7, so the four lanes of a row cover 32
// consecutive inputs a word and every group size from 32 on ends between
// words.  Inside a word, codes 2 j and 2 j + 1 sit 16 bits apart at bit 4 j:
// one shift, mask and or makes them a pair of 16-bit floats.  Scales: [tile]
// [group][16 rows].  Codes behind the last input or output are 8 (zero).
struct trba_linear_int4 {
    int in = 0, out = 0, group = 0, groups = 0, device = 0, scale_dtype = 0;
    int tiles = 0, chunks = 0;
    int gpc = 0;                // groups a chunk touches (1 for groups of 128 and more)
    int groups_pad = 0;         // groups a tile has room for
    uint8_t *base = nullptr;    // one allocation: codes, scales, bias
    uint8_t *codes = nullptr;   // [tiles][chunks][1024]
    uint8_t *scales = nullptr;  // [tiles][groups_pad][16] f32 or f16
    float *bias = nullptr;      // [out]
};

namespace trba {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// One warp a group: scale = max |w| / 7, code = 8 + round(w / scale).
__global__ void __launch_bounds__(256) int4_quantize_kernel(const float *__restrict__ w, int in, int out, int group,
                                                            int groups, uint8_t *__restrict__ codes, i64 pitch,
                                                            float *__restrict__ scales) {
    const int lane = threadIdx.x & 31;
    const i64 total = (i64)out * groups, step = (i64)gridDim.x * (blockDim.x >> 5);
    for (i64 e = (i64)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); e < total; e += step) {
        const i64 n = e / groups;
        const int k0 = (int)(e - n * groups) * group, k1 = min(in, k0 + group);
        const float *row = w + n * in;
        float mx = 0.0f;
        for (int k = k0 + lane; k < k1; k += 32) mx = fmaxf(mx, fabsf(row[k]));
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
        const float s = mx > 0.0f ? fdiv(mx, 7.0f) : 1.0f;
        if (lane == 0) scales[e] = s;
        for (int k = k0 + 2 * lane; k < k1; k += 64) {
            unsigned byte = 0;
            for (int h = 0; h < 2; ++h) {
                const float v = k + h < k1 ? fminf(fmaxf(fdiv(row[k + h], s), -7.0f), 7.0f) : 0.0f;
                byte |= (unsigned)((int)roundf(v) + 8) << (4 * h);
            }
            codes[n * pitch + (k >> 1)] = (uint8_t)byte;
        }
    }
}

// Natural codes [out][pitch] and scales [out][groups] -> the layout above, one
// thread a 4-byte word of codes and one a scale.
template <class S>
__global__ void __launch_bounds__(256) int4_layout_kernel(const uint8_t *__restrict__ codes, i64 pitch,
                                                          const S *__restrict__ scales, i64 ld_scales, int in, int out,
                                                          int groups, int groups_pad, int tiles, int chunks,
                                                          uint32_t *__restrict__ words, S *__restrict__ dst) {
    const i64 n_words = (i64)tiles * chunks * 256, n_scales = (i64)tiles * groups_pad * 16;
    GRID_LOOP(e, n_words + n_scales) {
        if (e < n_words) {
            const int w = (int)(e & 3), l = (int)(e >> 2) & 31, half = (int)(e >> 7) & 1;
            const i64 block = e >> 8, tile = block / chunks;
            const int n = (int)tile * 16 + half * 8 + (l >> 2);
            const int k0 = (int)(block - tile * chunks) * 128 + w * 32 + (l & 3) * 8;
            uint32_t v = 0;
            for (int c = 0; c < 8; ++c) {
                const int k = k0 + c;
                const uint32_t q = n < out && k < in ? (codes[n * pitch + (k >> 1)] >> (4 * (k & 1))) & 15u : 8u;
                v |= q << (4 * (c >> 1) + 16 * (c & 1));
            }
            words[e] = v;
        } else {
            const i64 f = e - n_words, tg = f >> 4, tile = tg / groups_pad;
            const int n = (int)tile * 16 + (int)(f & 15), g = (int)(tg - tile * groups_pad);
            dst[f] = n < out && g < groups ? scales[n * ld_scales + g] : S(0.0f);
        }
    }
}

// The reverse, for the host copies of the state.
__global__ void __launch_bounds__(256) int4_natural_kernel(const uint32_t *__restrict__ words, int in, int out,
                                                           int chunks, uint8_t *__restrict__ codes) {
    const int pitch = (int)(((i64)in + 1) / 2);
    GRID_LOOP(e, (i64)out * pitch) {
        const i64 n = e / pitch;
        const int k = (int)(e - n * pitch) * 2;
        const int half = (int)(n >> 3) & 1, l = (int)(n & 7) * 4 + ((k >> 3) & 3), w = (k >> 5) & 3;
        const uint32_t v = words[(((n >> 4) * chunks + (k >> 7)) * 2 + half) * 128 + l * 4 + w];
        const int c = k & 7;
        codes[e] = (uint8_t)(((v >> (2 * c)) & 15u) | (((v >> (2 * c + 16)) & 15u) << 4));
    }
}

// ----------------------------------------------------------------- forward --
constexpr int kDepth = 6;  // stages of a warp's ring

// y^T = W x^T on the tensor cores: A is a 16-output tile of the weights, the
// codes turned into exact bf16 or f16 integers in registers, B the
// activations from shared memory, eight columns at a time.  An f32
// activation enters as three bf16 columns whose sum it is exactly, so its
// products with the codes are exact in all types, and a group's sum is
// accumulated in f32 before its scale multiplies it.
//
// What bounds it: at few rows, reading the codes (half a byte a weight).  The
// warp-level mma is enough for that: a 1 KB block of codes costs 8 mma per
// eight columns and about 90 integer and conversion instructions.
//
// One CTA a SM for the whole product: its tiles are a contiguous share of all
// of them, its warps are `wn` units of MT tiles by `wk` interleaved parts of
// the inputs.  Every warp streams its blocks, over all its tiles, through a
// ring of cp.async stages of its own, so that loads stay in flight while
// activations are staged, sums are joined and outputs written.  Activations
// are staged in slabs of inputs, each once a CTA, all tiles running over one
// slab before the next; sums wait in shared memory in between.  The order of
// every sum is fixed.
struct Args {
    const uint8_t *codes, *scales;
    const float *bias;
    const void *x;
    void *y;
    i64 ldx, ldy;
    int in, out, rows, dtype;
    int tiles, chunks, gpc, groups_pad, scale_f16;
    int cpg;             // chunks a group has (1 for groups of up to 128)
    int wn;              // wk = warps / wn
    int slab;            // chunks whose activations are staged at once
    int block_rows;      // rows a CTA takes
    int packed;          // f32: columns 3 r + p of a single column tile (else p * rows + r)
    int xs_at, red_at, sums_at;  // shared memory: ring, activations, partial sums, sums between slabs
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
    const float z0 = first ? 0.0f : c[0], z1 = first ? 0.0f : c[1], z2 = first ? 0.0f : c[2], z3 = first ? 0.0f : c[3];
    if (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
}

// Codes at bits 4 j and 4 j + 16 of a word as a pair of floats, code - 8: the
// code is or-ed into the mantissa of 128 (bf16) or 1024 (f16), where one step
// is 1, and 136 or 1032 is subtracted; both exact.
template <bool F16>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    uint32_t r;
    if (F16) {
        r = (w & 0x000f000fu) | 0x64006400u;
        const __half2 v = __hsub2(*reinterpret_cast<__half2 *>(&r), __half2half2(__ushort_as_half(0x6408)));
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    r = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v =
        __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&r), __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Eight f32 or 16-bit activations of one row, zero behind the last input.
struct Eight {
    uint4 lo, hi;  // 16-bit types use lo only
};
__device__ __forceinline__ Eight load8(const Args &a, i64 row, int k) {
    Eight v;
    v.lo = v.hi = make_uint4(0, 0, 0, 0);
    if (a.dtype != TRBA_F32) {
        const uint16_t *src = static_cast<const uint16_t *>(a.x) + row * a.ldx + k;
        if (k + 8 <= a.in && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            v.lo = *reinterpret_cast<const uint4 *>(src);
        } else if (k >= 8 && k + 16 <= a.in) {  // the two aligned blocks it lies in are all of this row
            const uintptr_t at = reinterpret_cast<uintptr_t>(src);
            const uint4 *p = reinterpret_cast<const uint4 *>(at & ~(uintptr_t)15);
            const uint4 q0 = p[0], q1 = p[1];
            const uint32_t w[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
            const int by = ((int)at & 15) >> 2, sh = ((int)at & 2) * 8;
            uint32_t s[5];
#pragma unroll
            for (int i = 0; i < 5; ++i)
                s[i] = by == 0 ? w[i] : by == 1 ? w[min(i + 1, 7)] : by == 2 ? w[min(i + 2, 7)] : w[min(i + 3, 7)];
            v.lo = make_uint4(__funnelshift_r(s[0], s[1], sh), __funnelshift_r(s[1], s[2], sh),
                              __funnelshift_r(s[2], s[3], sh), __funnelshift_r(s[3], s[4], sh));
        } else {
            uint16_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = k + i < a.in ? src[i] : (uint16_t)0;
            v.lo = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                              h[6] | (uint32_t)h[7] << 16);
        }
    } else {
        const uint32_t *src = static_cast<const uint32_t *>(a.x) + row * a.ldx + k;
        if (k + 8 <= a.in && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            v.lo = reinterpret_cast<const uint4 *>(src)[0];
            v.hi = reinterpret_cast<const uint4 *>(src)[1];
        } else {
            uint32_t f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = k + i < a.in ? src[i] : 0u;
            v.lo = make_uint4(f[0], f[1], f[2], f[3]);
            v.hi = make_uint4(f[4], f[5], f[6], f[7]);
        }
    }
    return v;
}

// Stores them as one 16-bit column, or as three bf16 columns, `apart` bytes
// from each other, that add up to the f32 values: truncated to 8 bits three
// times (an infinity or NaN goes into the first alone).
__device__ __forceinline__ void store8(const Args &a, const Eight &v, uint8_t *dst, int apart) {
    if (a.dtype != TRBA_F32) {
        *reinterpret_cast<uint4 *>(dst) = v.lo;
        return;
    }
    const uint32_t f[8] = {v.lo.x, v.lo.y, v.lo.z, v.lo.w, v.hi.x, v.hi.y, v.hi.z, v.hi.w};
    uint32_t part[3][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = __uint_as_float(f[i]);
        const bool finite = fabsf(x) <= 3.402823466e38f;
        const uint32_t h = finite ? f[i] & 0xffff0000u : (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(x)) << 16;
        const float r1 = finite ? x - __uint_as_float(h) : 0.0f;
        const uint32_t m = __float_as_uint(r1) & 0xffff0000u;
        const uint32_t l = __float_as_uint(r1 - __uint_as_float(m)) & 0xffff0000u;
        const uint32_t q[3] = {h, m, l};
#pragma unroll
        for (int p = 0; p < 3; ++p) part[p][i >> 1] = i & 1 ? part[p][i >> 1] | q[p] : q[p] >> 16;
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
        *reinterpret_cast<uint4 *>(dst + p * apart) = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
}

// WG: words (32 inputs) a group has in a chunk; NT: tiles of eight columns;
// MT: tiles of 16 outputs a warp takes at once, so that it reads the
// activations from shared memory once for all of them; W: warps.
template <bool F16, int WG, int NT, int MT, int W>
__global__ void __launch_bounds__(W * 32, 1) int4_forward_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wk_n = W / a.wn, wn = warp / wk_n, wk = warp - wn * wk_n;
    const int units = (a.tiles + MT - 1) / MT;
    const int u0 = (int)((i64)units * blockIdx.x / gridDim.x) + wn;
    const int u1 = (int)((i64)units * (blockIdx.x + 1) / gridDim.x);
    const int row0 = blockIdx.y * a.block_rows, rows = min(a.block_rows, a.rows - row0);
    const int split = a.dtype == TRBA_F32 ? 3 : 1;
    const int es = a.scale_f16 ? 2 : 4, sb = 16 * a.gpc * es, part = 1024 + sb, slot = MT * part;
    const int pitch = a.slab * 256 + 64;  // 64 mod 128: eight lanes' 16-byte reads meet 32 different banks
    uint8_t *ring = smem + warp * kDepth * slot;
    uint8_t *xs = smem + a.xs_at;

    // the stream of this warp's blocks: for each slab, for each of its units, every wk_n-th chunk
    int pu = u0, pend = min(a.slab, a.chunks), pc = wk, pbase = 0;
    const uint8_t *psrc = a.codes, *pscale = a.scales;
    bool fresh = true;
    uint32_t dst = smem_addr(ring) + lane * 16;
    const uint32_t dst_end = dst + kDepth * slot;
    auto issue = [&]() {
        while (pc >= pend || pu >= u1) {
            if (pu < u1) {
                pu += a.wn;
            }
            if (pu >= u1) {
                if (pend >= a.chunks || u0 >= u1) {
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    return;
                }
                pu = u0;
                pbase = pend;
                pend = min(pend + a.slab, a.chunks);
            }
            pc = pbase + wk;
            fresh = true;
        }
        if (fresh) {
            psrc = a.codes + ((i64)pu * MT * a.chunks + pc) * 1024 + lane * 16;
            pscale = a.scales + (i64)pu * MT * a.groups_pad * 16 * es + lane * 16;
            fresh = false;
        }
        const int g = WG < 4 ? pc * (4 / WG) : a.cpg == 1 ? pc : pc / a.cpg;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (m && pu * MT + m >= a.tiles) break;  // (the sums of a tile that is not there are not stored)
            const uint8_t *p = psrc + (i64)m * a.chunks * 1024;
            cp16(dst + m * part, p);
            cp16(dst + m * part + 512, p + 512);
            if (lane * 16 < sb) cp16(dst + m * part + 1024, pscale + ((i64)m * a.groups_pad + g) * 16 * es);
        }
        psrc += wk_n * 1024;
        pc += wk_n;
        dst += slot;
        if (dst == dst_end) dst -= kDepth * slot;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kDepth - 1; ++i) issue();

    const int g = lane >> 2, t = lane & 3;
    // a column of mma depends on its own activations alone: lanes behind the
    // last column read it again
    const uint8_t *xcol[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        int col = n * 8 + g;
        if (split == 1 || a.packed) {
            col = min(col, rows * split - 1);
        } else {
            constexpr int kPer = (NT + 2) / 3;
            col = (n / kPer) * rows + min((n % kPer) * 8 + g, rows - 1);
        }
        xcol[n] = xs + col * pitch + t * 16;
    }
    const uint8_t *blk = ring;
    int turn = 0;  // partial-sum buffers are used in turn
    for (int s0 = 0; s0 < a.chunks; s0 += a.slab) {
        const int sc = min(a.slab, a.chunks - s0), n8 = sc * 16;
        if (s0) __syncthreads();
        // four loads in flight a thread
        for (int e0 = threadIdx.x; e0 < rows * n8; e0 += 4 * W * 32) {
            Eight v[4];
            int r[4], k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int e = e0 + u * W * 32;
                r[u] = e / n8, k[u] = e - r[u] * n8;
                if (r[u] < rows) v[u] = load8(a, row0 + r[u], s0 * 128 + k[u] * 8);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (r[u] < rows)
                    store8(a, v[u], xs + (a.packed ? 3 * r[u] : r[u]) * pitch + k[u] * 16,
                           a.packed ? pitch : rows * pitch);
        }
        __syncthreads();
        for (int u = u0; u < u1; u += a.wn, turn ^= 1) {
            float tot[MT][NT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) tot[m][n][0] = tot[m][n][1] = tot[m][n][2] = tot[m][n][3] = 0.0f;
            for (int ck = wk; ck < sc; ck += wk_n) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
                __syncwarp();
                issue();
                const int xo = ck * 256;
                uint32_t wl[MT][4], wh[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint4 lo = *reinterpret_cast<const uint4 *>(blk + m * part + lane * 16);
                    const uint4 hi = *reinterpret_cast<const uint4 *>(blk + m * part + 512 + lane * 16);
                    wl[m][0] = lo.x, wl[m][1] = lo.y, wl[m][2] = lo.z, wl[m][3] = lo.w;
                    wh[m][0] = hi.x, wh[m][1] = hi.y, wh[m][2] = hi.z, wh[m][3] = hi.w;
                }
                float c[MT][NT][4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t a0[MT][4], a1[MT][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        a0[m][0] = code_pair<F16>(wl[m][w]), a0[m][1] = code_pair<F16>(wh[m][w]);
                        a0[m][2] = code_pair<F16>(wl[m][w] >> 4), a0[m][3] = code_pair<F16>(wh[m][w] >> 4);
                        a1[m][0] = code_pair<F16>(wl[m][w] >> 8), a1[m][1] = code_pair<F16>(wh[m][w] >> 8);
                        a1[m][2] = code_pair<F16>(wl[m][w] >> 12), a1[m][3] = code_pair<F16>(wh[m][w] >> 12);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 b = *reinterpret_cast<const uint4 *>(xcol[n] + xo + w * 64);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            mma<F16>(c[m][n], a0[m], b.x, b.y, w % WG == 0);
                            mma<F16>(c[m][n], a1[m], b.z, b.w, false);
                        }
                    }
                    if (w % WG == WG - 1) {
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            float s0f, s1f;
                            const uint8_t *sp = blk + m * part + 1024 + (w / WG) * 16 * es;
                            if (a.scale_f16) {
                                s0f = __half2float(reinterpret_cast<const __half *>(sp)[g]);
                                s1f = __half2float(reinterpret_cast<const __half *>(sp)[g + 8]);
                            } else {
                                s0f = reinterpret_cast<const float *>(sp)[g];
                                s1f = reinterpret_cast<const float *>(sp)[g + 8];
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                tot[m][n][0] = fmaf(s0f, c[m][n][0], tot[m][n][0]);
                                tot[m][n][1] = fmaf(s0f, c[m][n][1], tot[m][n][1]);
                                tot[m][n][2] = fmaf(s1f, c[m][n][2], tot[m][n][2]);
                                tot[m][n][3] = fmaf(s1f, c[m][n][3], tot[m][n][3]);
                            }
                        }
                    }
                }
                blk += slot;
                if (blk == ring + kDepth * slot) blk = ring;
            }
            // join the wk_n warps of the unit; two buffers in turn, so that a
            // buffer is written again only after the next unit's barrier
            constexpr int kFrag = MT * NT;  // float4 of a lane
            if (wk_n > 1) {
                float4 *red = reinterpret_cast<float4 *>(smem + a.red_at) +
                              ((i64)(turn * a.wn + wn) * (wk_n - 1)) * kFrag * 32 + lane;
                if (wk > 0) {
#pragma unroll
                    for (int f = 0; f < kFrag; ++f) {
                        const float *v = tot[f / NT][f % NT];
                        red[((wk - 1) * kFrag + f) * 32] = make_float4(v[0], v[1], v[2], v[3]);
                    }
                }
                asm volatile("bar.sync %0, %1;" ::"r"(1 + wn), "r"(wk_n * 32) : "memory");
                if (wk > 0) continue;
                for (int k = 0; k < wk_n - 1; ++k)
#pragma unroll
                    for (int f = 0; f < kFrag; ++f) {
                        const float4 v = red[(k * kFrag + f) * 32];
                        float *o = tot[f / NT][f % NT];
                        o[0] += v.x, o[1] += v.y, o[2] += v.z, o[3] += v.w;
                    }
            }
            if (a.slab < a.chunks) {
                float4 *sums = reinterpret_cast<float4 *>(smem + a.sums_at) + (i64)(u - (u0 - wn)) * kFrag * 32 + lane;
#pragma unroll
                for (int f = 0; f < kFrag; ++f) {
                    float *o = tot[f / NT][f % NT];
                    if (s0) {
                        const float4 v = sums[f * 32];
                        o[0] += v.x, o[1] += v.y, o[2] += v.z, o[3] += v.w;
                    }
                    if (s0 + sc < a.chunks) sums[f * 32] = make_float4(o[0], o[1], o[2], o[3]);
                }
                if (s0 + sc < a.chunks) continue;
            }
            // outputs u * MT * 16 + 16 m + g and + 8 of the rows in this lane's columns
            auto put = [&](int r, int n, float v) {
                if (r >= rows || n >= a.out) return;
                v += a.bias[n];
                const i64 at = (row0 + r) * a.ldy + n;
                if (a.dtype == TRBA_F32) static_cast<float *>(a.y)[at] = v;
                else if (a.dtype == TRBA_BF16) static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(v);
                else static_cast<__half *>(a.y)[at] = __float2half_rn(v);
            };
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int n0 = (u * MT + m) * 16 + g;
                if (split == 1) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int q = 0; q < 4; ++q) put(n * 8 + 2 * t + (q & 1), n0 + (q >> 1) * 8, tot[m][n][q]);
                } else if (NT == 1) {  // packed: columns 3 r, 3 r + 1, 3 r + 2 lie in up to two lanes
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            float v[3];
#pragma unroll
                            for (int p = 0; p < 3; ++p)
                                v[p] = __shfl_sync(kFull, tot[m][0][2 * h + ((3 * r + p) & 1)], 4 * g + (3 * r + p) / 2);
                            if (t == r) put(r, n0 + 8 * h, v[0] + (v[1] + v[2]));
                        }
                } else if (NT % 3 == 0) {
#pragma unroll
                    for (int n = 0; n < NT / 3; ++n)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            put(n * 8 + 2 * t + (q & 1), n0 + (q >> 1) * 8,
                                tot[m][n][q] + (tot[m][n + NT / 3][q] + tot[m][n + 2 * (NT / 3)][q]));
                }
            }
        }
    }
}

int launched() {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
    return (int)e;
}

constexpr int kMaxSmem = 227 * 1024;
constexpr int kMaxJoin = 48 * 1024;  // shared memory of the warps' partial sums

template <bool F16, int WG, int NT, int MT, int W>
int launch(const Args &a, dim3 grid, size_t smem, cudaStream_t st) {
    auto fn = int4_forward_kernel<F16, WG, NT, MT, W>;
    static std::atomic<unsigned long long> sized{0};  // one bit a device: its limit has been raised
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(sized.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(fn),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) {
            report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
            return (int)e;
        }
        sized.fetch_or(bit, std::memory_order_relaxed);
    }
    fn<<<grid, W * 32, smem, st>>>(a);
    return launched();
}

template <bool F16, int WG>
int launch_nt(const Args &a, int nt, dim3 grid, size_t smem, cudaStream_t st) {
    switch (nt) {
        case 1: return launch<F16, WG, 1, 1, 16>(a, grid, smem, st);
        case 2: return launch<F16, WG, 2, 1, 16>(a, grid, smem, st);
        case 3: return launch<F16, WG, 3, 2, 8>(a, grid, smem, st);
        case 4: return launch<F16, WG, 4, 2, 8>(a, grid, smem, st);
        case 5: return launch<F16, WG, 5, 2, 8>(a, grid, smem, st);
        case 6: return launch<F16, WG, 6, 2, 8>(a, grid, smem, st);
        default: return launch<F16, WG, 8, 2, 8>(a, grid, smem, st);
    }
}

int forward(const trba_linear_int4 *l, const void *x, int dtype, i64 ldx, int rows, void *y, i64 ldy, cudaStream_t st) {
    Args a{};
    a.codes = l->codes, a.scales = l->scales, a.bias = l->bias;
    a.x = x, a.y = y, a.ldx = ldx, a.ldy = ldy;
    a.in = l->in, a.out = l->out, a.rows = rows, a.dtype = dtype;
    a.tiles = l->tiles, a.chunks = l->chunks, a.gpc = l->gpc;
    a.cpg = l->group >= 128 ? l->group / 128 : 1;
    a.groups_pad = l->groups_pad, a.scale_f16 = l->scale_dtype == TRBA_F16;
    // rows of a CTA: up to 64 columns, an f32 row being three (16 rows make six tiles of them)
    const bool f32 = dtype == TRBA_F32;
    const int most = f32 ? 16 : 64, blocks_y = (rows + most - 1) / most;
    a.block_rows = (rows + blocks_y - 1) / blocks_y;
    a.packed = f32 && a.block_rows <= 2;
    int nt = f32 ? (a.packed ? 1 : a.block_rows <= 8 ? 3 : 6) : (a.block_rows + 7) / 8;
    if (nt == 7) nt = 8;
    const int mt = nt <= 2 ? 1 : 2, warps = nt <= 2 ? 16 : 8;
    const int cols = a.block_rows * (f32 ? 3 : 1);
    i64 smem = 0;
    const int units = (a.tiles + mt - 1) / mt;
    const int frag = mt * nt * 512;  // bytes of one unit's sums
    const int ring = warps * kDepth * mt * (1024 + 16 * a.gpc * (a.scale_f16 ? 2 : 4));
    const auto x_bytes = [&](int chunks) { return ((i64)cols * (chunks * 256 + 64) + 127) & ~127ll; };
    int ctas = units < sm_count() ? units : sm_count();
    for (;; ctas = ctas * 2 < units ? ctas * 2 : units) {
        const int share = (units + ctas - 1) / ctas;  // units of a CTA, at most
        // Units of a CTA that run side by side: the fewest steps of (chunks a
        // warp streams + the join of the warps that share a unit).
        long long best = -1;
        int red = 0;
        for (int wn = warps; wn >= 1; wn >>= 1) {
            const int wk = warps / wn, bytes = 2 * wn * (wk - 1) * frag;
            const long long steps = (share + wn - 1) / wn;
            const long long cost = steps * (4 * ((a.chunks + wk - 1) / wk) + (wk > 1 ? 4 + wk : 0));
            if (bytes <= kMaxJoin && (best < 0 || cost < best)) best = cost, a.wn = wn, red = bytes;
        }
        if (const char *e = getenv("TUNE_WN")) a.wn = atoi(e), red = 2 * a.wn * (warps / a.wn - 1) * frag;
        // All activations at once where they fit; else as many chunks as fit
        // beside the sums that wait between slabs.  Sums that leave no room
        // for a slab of a few chunks go to more CTAs.
        const i64 room = kMaxSmem - ring - red;
        i64 sums = 0;
        a.slab = a.chunks;
        if (x_bytes(a.chunks) > room) {
            sums = (i64)share * frag;
            a.slab = (int)(((room - sums - 128) / cols - 64) / 256);
            if (a.slab < 4 && ctas < units) continue;
        }
        if (const char *e = getenv("TUNE_SLAB")) a.slab = atoi(e), sums = (i64)share * frag;
        a.xs_at = ring;
        a.red_at = a.xs_at + (int)x_bytes(a.slab);
        a.sums_at = a.red_at + red;
        smem = a.sums_at + sums;
        break;
    }
    const int wg = l->group >= 128 ? 4 : l->group / 32;
    const dim3 grid(ctas, blocks_y);
    if (dtype == TRBA_F16) {
        if (wg == 1) return launch_nt<true, 1>(a, nt, grid, smem, st);
        if (wg == 2) return launch_nt<true, 2>(a, nt, grid, smem, st);
        return launch_nt<true, 4>(a, nt, grid, smem, st);
    }
    if (wg == 1) return launch_nt<false, 1>(a, nt, grid, smem, st);
    if (wg == 2) return launch_nt<false, 2>(a, nt, grid, smem, st);
    return launch_nt<false, 4>(a, nt, grid, smem, st);
}

template <class S>
int layout(trba_linear_int4 *l, const uint8_t *codes, i64 pitch, const void *scales, i64 ld_scales, cudaStream_t st) {
    const i64 n = (i64)l->tiles * l->chunks * 256 + (i64)l->tiles * l->groups_pad * 16;
    int4_layout_kernel<S><<<grid_for(n), 256, 0, st>>>(codes, pitch, static_cast<const S *>(scales), ld_scales, l->in,
                                                       l->out, l->groups, l->groups_pad, l->tiles, l->chunks,
                                                       reinterpret_cast<uint32_t *>(l->codes),
                                                       reinterpret_cast<S *>(l->scales));
    return launched();
}

bool sizes_ok(int in, int out, int group) {
    return in > 0 && out > 0 && (group == 32 || group == 64 || (group >= 128 && group % 128 == 0));
}

trba_linear_int4 *allocate(int in, int out, int group, int scale_dtype) {
    auto *l = new (std::nothrow) trba_linear_int4;
    if (!l) return nullptr;
    l->in = in, l->out = out, l->group = group, l->groups = (in - 1) / group + 1;
    l->scale_dtype = scale_dtype;
    l->tiles = (out - 1) / 16 + 1;
    l->chunks = (in - 1) / 128 + 1;
    l->gpc = group >= 128 ? 1 : 128 / group;
    l->groups_pad = group >= 128 ? l->groups : l->chunks * l->gpc;
    const size_t nc = (size_t)l->tiles * l->chunks * 1024;
    const size_t ns = (size_t)l->tiles * l->groups_pad * 16 * (scale_dtype == TRBA_F32 ? 4 : 2);
    if (cudaGetDevice(&l->device) != cudaSuccess ||
        cudaMalloc(&l->base, nc + ns + (size_t)out * 4) != cudaSuccess) {
        cudaGetLastError();
        report_error(__FILE__, __LINE__, "LinearInt4: device allocation failed", -1);
        delete l;
        return nullptr;
    }
    l->codes = l->base;
    l->scales = l->base + nc;
    l->bias = reinterpret_cast<float *>(l->base + nc + ns);
    return l;
}

}  // namespace
}  // namespace trba

using namespace trba;

extern "C" {

trba_linear_int4 *trba_linear_int4_create(int in_features, int out_features, int group, const float *weight_f32,
                                          const float *bias) {
    TRBA_REQUIRE_RET(sizes_ok(in_features, out_features, group) && weight_f32, "trba_linear_int4_create: bad arguments",
                     nullptr);
    trba_linear_int4 *l = allocate(in_features, out_features, group, TRBA_F32);
    if (!l) return nullptr;
    const size_t nw = (size_t)in_features * out_features, ns = (size_t)out_features * l->groups;
    const i64 pitch = (in_features + 1ll) / 2;
    float *w = nullptr;  // the weights, then the scales, then the codes in their natural order
    bool ok = cudaMalloc(&w, (nw + ns) * 4 + (size_t)out_features * pitch) == cudaSuccess &&
              cudaMemcpy(w, weight_f32, nw * 4, cudaMemcpyHostToDevice) == cudaSuccess;
    ok = ok && (bias ? cudaMemcpy(l->bias, bias, (size_t)out_features * 4, cudaMemcpyHostToDevice)
                     : cudaMemset(l->bias, 0, (size_t)out_features * 4)) == cudaSuccess;
    if (ok) {
        float *scales = w + nw;
        uint8_t *codes = reinterpret_cast<uint8_t *>(scales + ns);
        int4_quantize_kernel<<<grid_for((i64)ns * 32), 256>>>(w, in_features, out_features, group, l->groups, codes,
                                                              pitch, scales);
        ok = launched() == 0 && layout<float>(l, codes, pitch, scales, l->groups, nullptr) == 0 &&
             cudaStreamSynchronize(nullptr) == cudaSuccess;
    }
    if (w) cudaFree(w);
    if (!ok) {
        report_error(__FILE__, __LINE__, "trba_linear_int4_create: allocation, copy or quantisation failed", -1);
        trba_linear_int4_destroy(l);
        return nullptr;
    }
    return l;
}

trba_linear_int4 *trba_linear_int4_create_codes(int in_features, int out_features, int group, const uint8_t *codes,
                                                long long ld_codes, const void *scales, int scale_dtype,
                                                long long ld_scales, const float *bias, void *stream) {
    TRBA_REQUIRE_RET(sizes_ok(in_features, out_features, group) && codes && scales &&
                         (scale_dtype == TRBA_F32 || scale_dtype == TRBA_F16) && ld_codes >= (in_features + 1ll) / 2 &&
                         ld_scales >= (in_features - 1) / group + 1,
                     "trba_linear_int4_create_codes: bad arguments", nullptr);
    trba_linear_int4 *l = allocate(in_features, out_features, group, scale_dtype);
    if (!l) return nullptr;
    cudaStream_t st = as_stream(stream);
    bool ok = (scale_dtype == TRBA_F16 ? layout<__half>(l, codes, ld_codes, scales, ld_scales, st)
                                       : layout<float>(l, codes, ld_codes, scales, ld_scales, st)) == 0;
    ok = ok && (bias ? cudaMemcpyAsync(l->bias, bias, (size_t)out_features * 4, cudaMemcpyDeviceToDevice, st)
                     : cudaMemsetAsync(l->bias, 0, (size_t)out_features * 4, st)) == cudaSuccess;
    if (cudaStreamSynchronize(st) != cudaSuccess) ok = false;
    if (!ok) {
        report_error(__FILE__, __LINE__, "trba_linear_int4_create_codes: copying the weights failed", -1);
        trba_linear_int4_destroy(l);
        return nullptr;
    }
    return l;
}

void trba_linear_int4_destroy(trba_linear_int4 *l) {
    if (!l) return;
    cudaFree(l->base);
    delete l;
}

int trba_linear_int4_forward(const trba_linear_int4 *l, const void *x, int dtype, long long ldx, int rows, void *y,
                             long long ldy, void *stream) {
    TRBA_REQUIRE_RET(l && rows >= 0 && rows <= (1 << 20), "trba_linear_int4_forward: bad arguments", -1);
    if (rows == 0) return 0;
    TRBA_REQUIRE_RET(x && y && ldx >= l->in && ldy >= l->out, "trba_linear_int4_forward: bad arguments", -1);
    TRBA_REQUIRE_RET(dtype == TRBA_F32 || dtype == TRBA_BF16 || dtype == TRBA_F16,
                     "trba_linear_int4_forward: unknown element type", -1);
    const uintptr_t es = dtype == TRBA_F32 ? 4 : 2;
    TRBA_REQUIRE_RET(reinterpret_cast<uintptr_t>(x) % es == 0 && reinterpret_cast<uintptr_t>(y) % es == 0,
                     "trba_linear_int4_forward: x or y is not aligned to its elements", -1);
    int dev = -1;
    cudaGetDevice(&dev);
    TRBA_REQUIRE_RET(dev == l->device, "trba_linear_int4_forward: the layer is on another device", -1);
    return forward(l, x, dtype, ldx, rows, y, ldy, as_stream(stream));
}

int trba_linear_int4_get(const trba_linear_int4 *l, uint8_t *codes, float *scales, float *bias) {
    if (!l) return -1;
    cudaError_t e = cudaDeviceSynchronize();
    if (codes && e == cudaSuccess) {
        const size_t n = (size_t)l->out * (((size_t)l->in + 1) / 2);
        uint8_t *nat = nullptr;
        e = cudaMalloc(&nat, n);
        if (e == cudaSuccess) {
            int4_natural_kernel<<<grid_for((i64)n), 256>>>(reinterpret_cast<const uint32_t *>(l->codes), l->in, l->out,
                                                           l->chunks, nat);
            e = (cudaError_t)launched();
            if (e == cudaSuccess) e = cudaMemcpy(codes, nat, n, cudaMemcpyDeviceToHost);
            cudaFree(nat);
        }
    }
    if (bias && e == cudaSuccess) e = cudaMemcpy(bias, l->bias, (size_t)l->out * 4, cudaMemcpyDeviceToHost);
    if (scales && e == cudaSuccess) {
        const bool f16 = l->scale_dtype == TRBA_F16;
        const size_t ns = (size_t)l->tiles * l->groups_pad * 16;
        uint8_t *tmp = new (std::nothrow) uint8_t[ns * (f16 ? 2 : 4)];
        TRBA_REQUIRE_RET(tmp, "trba_linear_int4_get: out of host memory", -1);
        e = cudaMemcpy(tmp, l->scales, ns * (f16 ? 2 : 4), cudaMemcpyDeviceToHost);
        for (int n = 0; n < l->out; ++n)
            for (int g = 0; g < l->groups; ++g) {
                const size_t at = ((size_t)(n >> 4) * l->groups_pad + g) * 16 + (n & 15);
                scales[(size_t)n * l->groups + g] = f16 ? __half2float(reinterpret_cast<const __half *>(tmp)[at])
                                                        : reinterpret_cast<const float *>(tmp)[at];
            }
        delete[] tmp;
    }
    if (e != cudaSuccess) report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
    return (int)e;
}

long long trba_linear_int4_param_count(const trba_linear_int4 *l) {
    return l ? (long long)l->in * l->out + l->out : -1;
}

}  // extern "C"
