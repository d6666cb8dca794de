// Linear layer with 4-bit weights and group scales for the few rows of a
// decoding step (include/trba_ops.h, LinearInt4).  No counterpart in the
// reference; the quantisation rule is LinearInt8's (src/linear.rs:53-59) for
// 4 bits and groups.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <new>

#include "common.cuh"
#include "trba_decode.h"
#include "trba_ops.h"

// Weight layout, made once when a layer is created: outputs in tiles of 16,
// inputs in chunks of 128, so that a warp streams one tile's chunks as
// consecutive blocks whose 16-byte pieces are already the A fragments of
// mma.m16n8k16.  A block is 1 KB of codes and the scales of its 16 rows.  In
// the codes, lane l = 4 g + t has 16 bytes of row g (first 512 bytes) and 16
// of row g + 8; their word w holds the codes of inputs 32 w + 8 t .. + 7, so
// the four lanes of a row cover 32 consecutive inputs a word and every group
// size from 32 on ends between words.  Inside a word, codes 2 j and 2 j + 1
// sit 16 bits apart at bit 4 j: one shift, mask and or makes them a pair of
// 16-bit floats.  Scales: [128 / group][16 rows]; a group of several chunks
// has its scale once a chunk (at most 6% more to read), so that all blocks
// look the same.  Codes behind the last input or output are 8 (zero).
struct trba_linear_int4 {
    int in = 0, out = 0, group = 0, groups = 0, device = 0, scale_dtype = 0;
    int tiles = 0, chunks = 0;
    int gpc = 0;                // scales of a row in a chunk (1 for groups of 128 and more)
    int block = 0;              // bytes of a block: 1024 + 16 gpc scales
    bool owned = true;          // base is this layer's own allocation
    uint8_t *base = nullptr;    // blocks [tiles][chunks], bias
    float *bias = nullptr;      // [out]
};

namespace trba {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;

// One warp a group: scale = max |w| / 7, code = 8 + round(w / scale).  Runs
// once a layer; bound by reading the f32 weights twice.
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

// Natural codes [out][pitch] and scales [out][groups] -> the layout above: a
// warp a block, a lane 8 words of codes, then the scales.  Runs once a layer;
// each word is one read where the rows allow it.  Making a 16384 x 16384 layer
// takes 0.49 ms with the copies of its arguments.
template <class S>
__global__ void __launch_bounds__(256) int4_layout_kernel(const uint8_t *__restrict__ codes, i64 pitch,
                                                          const S *__restrict__ scales, i64 ld_scales, int in, int out,
                                                          int group, int groups, int gpc, int tiles, int chunks,
                                                          int block, uint8_t *__restrict__ dst) {
    const int lane = threadIdx.x & 31;
    const i64 step = (i64)gridDim.x * 8;
    for (i64 e = (i64)blockIdx.x * 8 + (threadIdx.x >> 5); e < (i64)tiles * chunks; e += step) {
        const i64 tile = e / chunks;
        const int chunk = (int)(e - tile * chunks);
        uint8_t *out_block = dst + e * block;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const i64 n = tile * 16 + half * 8 + (lane >> 2);
            uint32_t v[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int k0 = chunk * 128 + w * 32 + (lane & 3) * 8;
                uint32_t q = 0x88888888u;  // eight codes as they come, four bits each
                if (n < out && k0 < in) {
                    const uint8_t *src = codes + n * pitch + (k0 >> 1);
                    if (k0 + 8 <= in) {
                        q = (reinterpret_cast<uintptr_t>(src) & 3) == 0
                                ? *reinterpret_cast<const uint32_t *>(src)
                                : src[0] | (uint32_t)src[1] << 8 | (uint32_t)src[2] << 16 | (uint32_t)src[3] << 24;
                    } else {
                        for (int k = k0; k < in; ++k) {
                            const int c = k - k0;
                            q = (q & ~(15u << (4 * c))) | ((src[c >> 1] >> (4 * (c & 1))) & 15u) << (4 * c);
                        }
                    }
                }
                uint32_t even = q & 0x0f0f0f0fu, odd = (q >> 4) & 0x0f0f0f0fu;
                even = (even | even >> 4) & 0x00ff00ffu, odd = (odd | odd >> 4) & 0x00ff00ffu;
                v[w] = ((even | even >> 8) & 0xffffu) | (odd | odd >> 8) << 16;
            }
            reinterpret_cast<uint4 *>(out_block + half * 512)[lane] = make_uint4(v[0], v[1], v[2], v[3]);
        }
        for (int f = lane; f < gpc * 16; f += 32) {
            const i64 n = tile * 16 + (f & 15), g = ((i64)chunk * 128 + (i64)(f >> 4) * 32 * (4 / gpc)) / group;
            reinterpret_cast<S *>(out_block + 1024)[f] = n < out && g < groups ? scales[n * ld_scales + g] : S(0.0f);
        }
    }
}

// The reverse, for the host copies of the state.
__global__ void __launch_bounds__(256) int4_natural_kernel(const uint8_t *__restrict__ base, int in, int out,
                                                           int chunks, int block, uint8_t *__restrict__ codes) {
    const int pitch = (int)(((i64)in + 1) / 2);
    GRID_LOOP(e, (i64)out * pitch) {
        const i64 n = e / pitch;
        const int k = (int)(e - n * pitch) * 2;
        const int half = (int)(n >> 3) & 1, l = (int)(n & 7) * 4 + ((k >> 3) & 3), w = (k >> 5) & 3;
        const uint32_t v = reinterpret_cast<const uint32_t *>(base + ((n >> 4) * chunks + (k >> 7)) * block)[half * 128 + l * 4 + w];
        const int c = k & 7;
        codes[e] = (uint8_t)(((v >> (2 * c)) & 15u) | (((v >> (2 * c + 16)) & 15u) << 4));
    }
}

// ----------------------------------------------------------------- forward --
// Few columns: 16 warps with three stages of two blocks each keep 64 KB in
// flight a SM while they work on 32.  8 f16 rows through 16384 x 8192 take 31 us
// so and 37 with 32 warps and two stages (one row: 25 and 27); a fourth stage,
// or stages of one block, gain nothing.
constexpr int kPair = 2, kFewStages = 3;
constexpr int kFewWarps = 16, kManyWarps = 16;
// More columns, in tiles of eight: the stages of a step, and the blocks that a
// warp takes in one.  Four stages instead of three gain a little at 4 and 5
// tiles (16384 x 8192: 49.3 and 50.4 us at 32 rows, 53.6 and 54.3 at 40) and
// nothing at 2 and 6; at 3 and 8 they leave room for fewer warps side by side
// (50001 x 4099: 65.7 -> 76.3 us at 24 rows, 135 -> 163 at 64).  Two blocks a
// step halve the barriers: 31.5 us instead of 37.0 at 16 rows through 16384 x
// 8192, 65.7 instead of 71.9 at 24 through 50001 x 4099 (but 14.1 instead of
// 12.3 through 4096 x 4096); from 5 tiles on their fragments take the room (40
// rows through 50001 x 4099: 96 -> 107 us, 64: 135 -> 153; at 4 tiles 84 -> 78
// there and 14.4 -> 16.4 through 4096 x 4096).
constexpr int many_depth(int nt) { return nt > 3 && nt <= 5 ? 4 : 3; }
constexpr int many_blocks(int nt) { return nt <= 3 ? 2 : 1; }

// y^T = W x^T on the tensor cores: A is a 16-output tile of the weights, the
// codes turned into exact bf16 or f16 integers in registers, B the
// activations, eight columns at a time.  An f32 activation enters as three
// bf16 columns whose sum it is exactly (down to 2^-133, a bf16's last place),
// so its products with the codes are exact in all types, and a group's sum is
// accumulated in f32 before its scale multiplies it.
//
// What bounds it: at few rows, reading the codes (half a byte a weight) and
// turning them into floats.  The warp-level mma is enough for that: a 1 KB block
// of codes costs 8 mma per eight columns and about 75 integer and conversion
// instructions, which take as long as reading the block.  tcgen05 was not
// built, so not measured either: its weights, as floats, would pass through
// tensor memory on the way, a group's sum would need columns of its own to be
// scaled from, and its 128-row tiles would be one to eight columns wide at the
// rows of a decoding step.
//
// One CTA a SM for the whole product, its tiles a contiguous share of all of
// them, its warps `wn` tiles side by side by `wk` parts of the inputs.  The
// order of every sum is fixed.
struct Args {
    const uint8_t *blocks;
    const float *bias;
    const void *x;
    void *y;
    uint4 *frags;  // [row block][chunk][word][column tile][lane]
    i64 ldx, ldy;
    int in, out, rows, dtype;
    int tiles, chunks;
    int wn;              // wk = warps / wn
    int cs;              // many columns: CTAs that share a tile's chunks
    int slab;            // few columns: chunks whose activations are staged at once
    int block_rows;      // many columns: rows a CTA takes
    int xs_at, red_at, sums_at;  // in shared memory: activations, partial sums, sums between slabs
};

__device__ __forceinline__ float scale_f32(float v) { return v; }
__device__ __forceinline__ float scale_f32(__half v) { return __half2float(v); }
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

// (w & mask) | bits in one instruction (left to itself the compiler takes two)
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 v) { return *reinterpret_cast<const uint32_t *>(&v); }
__device__ __forceinline__ uint32_t bf162_bits(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t *>(&v); }

// The four pairs of a word (codes at bits 4 j and 4 j + 16) as floats, exact,
// with one shift a word.  Or-ing a small integer into the mantissa of a power of
// two, instead of converting it, is a published method (Kim et al., "Who Says
// Elephants Can't Run", 2022, for 4-bit weights in f16); the bf16 form is this
// file's own.
// f16: the code is or-ed into the mantissa of 1024 at either of two places,
// the upper one worth 16 times as much: code - 8.
// bf16 has room for one place behind 128.  The place above it needs no
// magic number: the bits of exponent 0 and of exponent 1 count in the same
// steps of 2^-133, so a code at bits 4 .. 7 is code * 2^-129 and times 2^127
// a quarter of itself.  All pairs come as (code - 8) / 4; kUnit undoes it.
template <bool F16>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t &p0, uint32_t &p1, uint32_t &p2, uint32_t &p3) {
    const uint32_t v = w >> 8;
    if (F16) {
        const __half2 low = __half2half2(__ushort_as_half(0x6408)),   // 1032
            sixteenth = __half2half2(__ushort_as_half(0x2c00)), high = __half2half2(__ushort_as_half(0xd480));  // -72
        const uint32_t q0 = and_or(w, 0x000f000fu, 0x64006400u), q1 = and_or(w, 0x00f000f0u, 0x64006400u);
        const uint32_t q2 = and_or(v, 0x000f000fu, 0x64006400u), q3 = and_or(v, 0x00f000f0u, 0x64006400u);
        p0 = half2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&q0), low));
        p1 = half2_bits(__hfma2(*reinterpret_cast<const __half2 *>(&q1), sixteenth, high));
        p2 = half2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&q2), low));
        p3 = half2_bits(__hfma2(*reinterpret_cast<const __half2 *>(&q3), sixteenth, high));
    } else {
        const __nv_bfloat162 quarter = __bfloat162bfloat162(__ushort_as_bfloat16(0x3e80)),
                             low = __bfloat162bfloat162(__ushort_as_bfloat16(0xc208)),    // -34
            up = __bfloat162bfloat162(__ushort_as_bfloat16(0x7f00)),                      // 2^127
            high = __bfloat162bfloat162(__ushort_as_bfloat16(0xc000));                    // -2
        const uint32_t q0 = and_or(w, 0x000f000fu, 0x43004300u), q1 = w & 0x00f000f0u;
        const uint32_t q2 = and_or(v, 0x000f000fu, 0x43004300u), q3 = v & 0x00f000f0u;
        p0 = bf162_bits(__hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&q0), quarter, low));
        p1 = bf162_bits(__hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&q1), up, high));
        p2 = bf162_bits(__hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&q2), quarter, low));
        p3 = bf162_bits(__hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&q3), up, high));
    }
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

// The activations as B fragments: a thread eight of a row (three 16-byte
// pieces for f32).  Columns go row by row, an f32 row's three next to each
// other; what stands in the columns behind the last does not matter.  2 to 4 us,
// bound by its launch; the weights of the next kernel load meanwhile.
__global__ void __launch_bounds__(256) int4_fragments_kernel(const __grid_constant__ Args a, int nt) {
    const int split = a.dtype == TRBA_F32 ? 3 : 1;
    const int row0 = blockIdx.y * a.block_rows, rows = min(a.block_rows, a.rows - row0);
    uint4 *frags = a.frags + (i64)blockIdx.y * a.chunks * 4 * nt * 32;
    GRID_LOOP(e, (i64)a.chunks * 4 * rows * 4) {
        const int t = (int)(e & 3);
        const i64 q = e >> 2, cw = q / rows;
        const int r = (int)(q - cw * rows);
        const Eight v = load8(a, row0 + r, (int)cw * 32 + t * 8);
        uint4 part[3];
        store8(a, v, reinterpret_cast<uint8_t *>(part), 16);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const int c = split * r + p;
            if (p < split) frags[(cw * nt + (c >> 3)) * 32 + (c & 7) * 4 + t] = part[p];
        }
    }
}

// One block: tot += scales * (codes - 8) . activations.  x(w, n): the B
// fragment of word w and column tile n.  S: type of the scales; WG: words (32
// inputs) a group has in a chunk; NT: tiles of eight columns.
template <bool F16, class S, int WG, int NT, class X>
__device__ __forceinline__ void block_product(const uint8_t *blk, X x, float (&tot)[NT][4], int lane) {
    const uint4 lo = *reinterpret_cast<const uint4 *>(blk + lane * 16);
    const uint4 hi = *reinterpret_cast<const uint4 *>(blk + 512 + lane * 16);
    const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
    const S *sp = reinterpret_cast<const S *>(blk + 1024) + (lane >> 2);
    float c[NT][4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t a0[4], a1[4];
        code_pairs<F16>(wl[w], a0[0], a0[2], a1[0], a1[2]);
        code_pairs<F16>(wh[w], a0[1], a0[3], a1[1], a1[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint4 b = x(w, n);
            mma<F16>(c[n], a0, b.x, b.y, w % WG == 0);
            mma<F16>(c[n], a1, b.z, b.w, false);
        }
        if (w % WG == WG - 1) {
            const float s0 = scale_f32(sp[(w / WG) * 16]), s1 = scale_f32(sp[(w / WG) * 16 + 8]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                tot[n][0] = fmaf(s0, c[n][0], tot[n][0]);
                tot[n][1] = fmaf(s0, c[n][1], tot[n][1]);
                tot[n][2] = fmaf(s1, c[n][2], tot[n][2]);
                tot[n][3] = fmaf(s1, c[n][3], tot[n][3]);
            }
        }
    }
}

// Writes a tile's sums: outputs 16 tile + g and + 8 of the rows in this lane's columns.
template <bool F16, int NT>
__device__ __forceinline__ void write_tile(const Args &a, int tile, int row0, int rows, const float (&tot)[NT][4],
                                           int lane) {
    constexpr float kUnit = F16 ? 1.0f : 4.0f;  // of the code pairs
    const int g = lane >> 2, t = lane & 3, n0 = tile * 16 + g;
    auto put = [&](int r, int n, float v) {
        if (r >= rows || n >= a.out) return;
        v = fmaf(v, kUnit, a.bias[n]);
        const i64 at = (row0 + r) * a.ldy + n;
        if (a.dtype == TRBA_F32) static_cast<float *>(a.y)[at] = v;
        else if (a.dtype == TRBA_BF16) static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(v);
        else static_cast<__half *>(a.y)[at] = __float2half_rn(v);
    };
    if (a.dtype != TRBA_F32) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) put(n * 8 + 2 * t + (q & 1), n0 + (q >> 1) * 8, tot[n][q]);
    } else {  // columns 3 r, 3 r + 1, 3 r + 2 lie in up to two lanes
#pragma unroll
        for (int r = 0; r < NT * 8 / 3; ++r) {
            if (r >= rows) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    const int c = 3 * r + p;
                    v[p] = __shfl_sync(kFull, tot[c / 8][2 * h + (c & 1)], 4 * g + (c & 7) / 2);
                }
                if (t == (r & 3)) put(r, n0 + 8 * h, v[0] + (v[1] + v[2]));
            }
        }
    }
}

// Up to eight columns: every warp streams its blocks, over all its tiles,
// through a ring of cp.async stages of its own, so that loads stay in flight
// while activations are staged, sums are joined and outputs written.
// Activations are staged in slabs of inputs, each once a CTA, all tiles
// running over one slab before the next; sums wait in shared memory in between.
// One bf16 row through 16384 x 16384, groups of 128: 31.5 us, 4.4 TB/s of codes
// and scales, 0.67 of a copy's rate; one f16 row through 16384 x 8192, groups of
// 32: 20 us.  In the first of these a CTA has seven tiles for eight pairs of
// warps, so an eighth of them has nothing to do; the others wait for their own
// rings, with data, tensor pipe (25%) and issue slots (57%) all below their
// limits.  Sharing out the tiles so that a CTA has all inputs of its outputs
// needs no sums in memory.
template <bool F16, class S, int WG>
__global__ void __launch_bounds__(kFewWarps * 32, 1) int4_few_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int W = kFewWarps, NT = 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wk_n = W / a.wn, wn = warp / wk_n, wk = warp - wn * wk_n;
    const int t0 = (int)((i64)a.tiles * blockIdx.x / gridDim.x) + wn;
    const int t1 = (int)((i64)a.tiles * (blockIdx.x + 1) / gridDim.x);
    const int rows = a.rows, split = a.dtype == TRBA_F32 ? 3 : 1;
    constexpr int kBlock = 1024 + 16 * (4 / WG) * (int)sizeof(S), kSlot = kPair * kBlock;
    const int pitch = a.slab * 256 + 64;  // 64 mod 128: eight lanes' 16-byte reads meet 32 different banks
    const int ring = warp * kFewStages * kSlot;    // offsets in shared memory

    // the stream of this warp's stages: for each slab, for each of its tiles, its part of the chunks
    int ptile = t0 - a.wn, pslab = t0 < t1 ? 0 : a.chunks, left = 0;
    const uint8_t *psrc = a.blocks;
    const uint32_t ring_s = smem_addr(smem) + ring + lane * 16;
    uint32_t dst = ring_s;
    auto issue = [&]() {
        while (left <= 0 && pslab < a.chunks) {  // the next tile, or the next slab's first
            ptile += a.wn;
            if (ptile >= t1) {
                ptile = t0;
                pslab += a.slab;
                if (pslab >= a.chunks) break;
            }
            const int sc = min(a.slab, a.chunks - pslab), c = pslab + sc * wk / wk_n;
            left = pslab + sc * (wk + 1) / wk_n - c;
            psrc = a.blocks + ((i64)ptile * a.chunks + c) * kBlock + lane * 16;
        }
        if (left > 0) {
            const int bytes = min(left, kPair) * kBlock;
#pragma unroll
            for (int j = 0; j < (kSlot + 511) / 512; ++j)
                if (lane * 16 < bytes - 512 * j) cp16(dst + 512 * j, psrc + 512 * j);
            psrc += kSlot;
            left -= kPair;
            dst = dst == ring_s + (kFewStages - 1) * kSlot ? ring_s : dst + kSlot;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < kFewStages - 1; ++i) issue();

    // a column of mma depends on its own activations alone: lanes behind the
    // last column read it again
    const int xcol = a.xs_at + min(lane >> 2, rows * split - 1) * pitch + (lane & 3) * 16;
    int blk = ring, turn = 0;  // partial-sum buffers are used in turn
    for (int s0 = 0; s0 < a.chunks; s0 += a.slab) {
        const int sc = min(a.slab, a.chunks - s0), n8 = sc * 16;
        if (s0) __syncthreads();
        constexpr int kLoads = 2;  // in flight a thread
        for (int e0 = threadIdx.x; e0 < rows * n8; e0 += kLoads * W * 32) {
            Eight v[kLoads];
            int r[kLoads], k[kLoads];
#pragma unroll
            for (int u = 0; u < kLoads; ++u) {
                const int e = e0 + u * W * 32;
                r[u] = e / n8, k[u] = e - r[u] * n8;
                if (r[u] < rows) v[u] = load8(a, r[u], s0 * 128 + k[u] * 8);
            }
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
                if (r[u] < rows) store8(a, v[u], smem + a.xs_at + split * r[u] * pitch + k[u] * 16, pitch);
        }
        __syncthreads();
        const int cb = sc * wk / wk_n, ce = sc * (wk + 1) / wk_n;
        for (int u = t0; u < t1; u += a.wn, turn ^= 1) {
            float tot[NT][4] = {};
            for (int xo = cb * 256; xo < ce * 256; xo += kPair * 256) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
                __syncwarp();
                issue();
#pragma unroll
                for (int p = 0; p < kPair; ++p) {
                    if (p && xo + 256 * p >= ce * 256) break;
                    block_product<F16, S, WG, NT>(
                        smem + blk + p * kBlock,
                        [&](int w, int) { return *reinterpret_cast<const uint4 *>(smem + xcol + xo + p * 256 + w * 64); },
                        tot, lane);
                }
                blk = blk == ring + (kFewStages - 1) * kSlot ? ring : blk + kSlot;
            }
            // join the wk_n warps of the tile; two buffers in turn, so that a
            // buffer is written again only after the next tile's barrier
            if (wk_n > 1) {
                float4 *red = reinterpret_cast<float4 *>(smem + a.red_at) + ((turn * a.wn + wn) * (wk_n - 1)) * 32 + lane;
                if (wk > 0) red[(wk - 1) * 32] = make_float4(tot[0][0], tot[0][1], tot[0][2], tot[0][3]);
                asm volatile("bar.sync %0, %1;" ::"r"(1 + wn), "r"(wk_n * 32) : "memory");
                if (wk > 0) continue;
                for (int k = 0; k < wk_n - 1; ++k) {
                    const float4 v = red[k * 32];
                    tot[0][0] += v.x, tot[0][1] += v.y, tot[0][2] += v.z, tot[0][3] += v.w;
                }
            }
            if (a.slab < a.chunks) {
                float4 *sums = reinterpret_cast<float4 *>(smem + a.sums_at) + (u - (t0 - wn)) * 32 + lane;
                if (s0) {
                    const float4 v = *sums;
                    tot[0][0] += v.x, tot[0][1] += v.y, tot[0][2] += v.z, tot[0][3] += v.w;
                }
                if (s0 + sc < a.chunks) {
                    *sums = make_float4(tot[0][0], tot[0][1], tot[0][2], tot[0][3]);
                    continue;
                }
            }
            write_tile<F16, NT>(a, u, 0, rows, tot, lane);
        }
    }
}

// More columns: the CTA moves in steps of a block or two a warp, `wn` tiles
// side by side and wk warps deep, through stages that hold the step's B fragments
// (read by all warps) and each warp's block.  Staging the activations as
// fragments in memory first makes their copies plain and aligned; per SM and
// step they are read once for wn tiles.  From about 24 columns on the tensor
// pipe's floor is above memory's (a 16 x 8 x 16 mma takes 2.4 cycles a SM).
// 40 f16 rows through 50001 x 4099, groups of 32: 95 us with the fragments, 1.3
// TB/s of codes and scales and 173 TFLOP/s; tensor pipe 37%, issue slots 48%: bound
// by the shared-memory reads and conversions between the barriers of a step (a
// warp has one tile of 16 outputs, and reads all fragments for it).  16 rows
// through 16384 x 8192: 32 to 35 us, 64 rows 76 to 80 us.  Beyond 64 columns a
// row block follows the other, each reading and unpacking the whole layer: 128
// rows 147 us, 512 rows 498 us.
template <bool F16, class S, int WG, int NT>
__global__ void __launch_bounds__(kManyWarps * 32, 1) int4_many_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int D = many_depth(NT), KS = many_blocks(NT), kBlock = 1024 + 16 * (4 / WG) * (int)sizeof(S);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wk_n = kManyWarps / a.wn, wn = warp / wk_n, wk = warp - wn * wk_n;
    const int groups = (a.tiles + a.wn - 1) / a.wn;
    const int rank = blockIdx.x % a.cs, bx = blockIdx.x / a.cs, gx = gridDim.x / a.cs;
    const int g0 = (int)((i64)groups * bx / gx), g1 = (int)((i64)groups * (bx + 1) / gx);
    const int cb = a.chunks * rank / a.cs, ce = a.chunks * (rank + 1) / a.cs;  // this CTA's chunks
    const int row0 = blockIdx.y * a.block_rows, rows = min(a.block_rows, a.rows - row0);
    const int deep = wk_n * KS, xbytes = deep * NT * 2048, stage = xbytes + kManyWarps * KS * kBlock;
    const uint8_t *frags = reinterpret_cast<const uint8_t *>(a.frags) + (i64)blockIdx.y * a.chunks * NT * 2048;
    const uint32_t smem_s = smem_addr(smem);
    float4 *red = reinterpret_cast<float4 *>(smem + a.red_at);

    int pg = g0, pc = cb, ps = 0;  // the next stage to fill: its group, first chunk, place
    auto weights = [&](uint32_t to) {
        const int tile = pg * a.wn + wn, c = pc + wk * KS;
        if (pg < g1 && tile < a.tiles && c < ce) {
            const uint8_t *src = a.blocks + ((i64)tile * a.chunks + c) * kBlock + lane * 16;
            const uint32_t dst = to + xbytes + warp * KS * kBlock + lane * 16;
            const int bytes = min(KS, ce - c) * kBlock - lane * 16;
#pragma unroll
            for (int o = 0; o < KS * kBlock; o += 512)
                if (o < bytes) cp16(dst + o, src + o);
        }
    };
    auto activations = [&](uint32_t to) {
        if (pg < g1) {
            const int bytes = min(deep, ce - pc) * NT * 2048;
            const uint8_t *src = frags + (i64)pc * NT * 2048;
            for (int o = threadIdx.x * 16; o < bytes; o += kManyWarps * 32 * 16) cp16(to + o, src + o);
        }
    };
    auto next = [&]() {
        pc += deep;
        if (pc >= ce) {
            pc = cb;
            ++pg;
        }
        ps = ps + 1 == D ? 0 : ps + 1;
    };
    // the first weights are on their way while the fragments are made
    weights(smem_s);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = 0; i < D - 1; ++i) {
        if (i) weights(smem_s + ps * stage);
        activations(smem_s + ps * stage);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next();
    }
    int cs = 0;
    for (int g = g0; g < g1; ++g) {
        const int tile = g * a.wn + wn;
        float tot[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) tot[n][0] = tot[n][1] = tot[n][2] = tot[n][3] = 0.0f;
        for (int c0 = cb; c0 < ce; c0 += deep) {
            asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
            __syncthreads();  // the stage is there for all, and the last one is free
            weights(smem_s + ps * stage);
            activations(smem_s + ps * stage);
            asm volatile("cp.async.commit_group;" ::: "memory");
            next();
            const uint8_t *st = smem + cs * stage;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                if (tile >= a.tiles || c0 + wk * KS + j >= ce) break;
                const uint8_t *xs = st + (wk * KS + j) * NT * 2048 + lane * 16;
                block_product<F16, S, WG, NT>(
                    st + xbytes + (warp * KS + j) * kBlock,
                    [&](int w, int n) { return *reinterpret_cast<const uint4 *>(xs + (w * NT + n) * 512); }, tot, lane);
            }
            cs = cs + 1 == D ? 0 : cs + 1;
        }
        // join the warps of a tile; the next group's first barrier keeps `red` until it was read
        if (wk_n > 1) {
            if (wk > 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    red[((wn * (wk_n - 1) + wk - 1) * NT + n) * 32 + lane] =
                        make_float4(tot[n][0], tot[n][1], tot[n][2], tot[n][3]);
            }
            __syncthreads();
            if (wk == 0) {
                for (int k = 0; k < wk_n - 1; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float4 v = red[((wn * (wk_n - 1) + k) * NT + n) * 32 + lane];
                        tot[n][0] += v.x, tot[n][1] += v.y, tot[n][2] += v.z, tot[n][3] += v.w;
                    }
            }
        }
        if (a.cs > 1) {  // one group a CTA: the stages are done with and hold the sums
            __syncthreads();
            float4 *part = reinterpret_cast<float4 *>(smem) + wn * NT * 32 + lane;
            if (rank > 0 && wk == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n) part[n * 32] = make_float4(tot[n][0], tot[n][1], tot[n][2], tot[n][3]);
            }
            cg::this_cluster().sync();
            if (rank == 0 && wk == 0) {
                for (int k = 1; k < a.cs; ++k) {
                    const float4 *other = cg::this_cluster().map_shared_rank(part, k);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float4 v = other[n * 32];
                        tot[n][0] += v.x, tot[n][1] += v.y, tot[n][2] += v.z, tot[n][3] += v.w;
                    }
                }
            }
            cg::this_cluster().sync();  // no CTA leaves while its sums are read
            if (rank > 0) return;
        }
        if (wk > 0) continue;
        if (tile < a.tiles) write_tile<F16, NT>(a, tile, row0, rows, tot, lane);
    }
}

int launched() {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
    return (int)e;
}

constexpr int kMaxSmem = 227 * 1024;

// Raises the kernel's shared-memory limit (once a device) and launches it;
// `overlap`: as soon as the kernel before it ends, its own wait taking care
// of the rest.
int launch(void (*fn)(const Args), std::atomic<unsigned long long> &sized, const Args &a, dim3 grid, int warps,
           size_t smem, bool overlap, cudaStream_t st) {
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
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cs, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = !overlap ? 0 : a.cs > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, fn, a);
    return launched();
}

template <bool F16, class S, int WG>
int launch_few(const Args &a, dim3 grid, size_t smem, cudaStream_t st) {
    static std::atomic<unsigned long long> sized{0};
    return launch(int4_few_kernel<F16, S, WG>, sized, a, grid, kFewWarps, smem, false, st);
}
template <bool F16, class S, int WG, int NT>
int launch_many(const Args &a, dim3 grid, size_t smem, cudaStream_t st) {
    static std::atomic<unsigned long long> sized{0};
    return launch(int4_many_kernel<F16, S, WG, NT>, sized, a, grid, kManyWarps, smem, true, st);
}

template <bool F16, class S, int WG>
int launch_nt(const Args &a, int nt, dim3 grid, size_t smem, cudaStream_t st) {
    switch (nt) {
        case 1: return launch_few<F16, S, WG>(a, grid, smem, st);
        case 2: return launch_many<F16, S, WG, 2>(a, grid, smem, st);
        case 3: return launch_many<F16, S, WG, 3>(a, grid, smem, st);
        case 4: return launch_many<F16, S, WG, 4>(a, grid, smem, st);
        case 5: return launch_many<F16, S, WG, 5>(a, grid, smem, st);
        case 6: return launch_many<F16, S, WG, 6>(a, grid, smem, st);
        default: return launch_many<F16, S, WG, 8>(a, grid, smem, st);
    }
}

template <bool F16>
int launch_type(const Args &a, bool scale_f16, int wg, int nt, dim3 grid, size_t smem, cudaStream_t st) {
    if (scale_f16) {
        if (wg == 1) return launch_nt<F16, __half, 1>(a, nt, grid, smem, st);
        if (wg == 2) return launch_nt<F16, __half, 2>(a, nt, grid, smem, st);
        return launch_nt<F16, __half, 4>(a, nt, grid, smem, st);
    }
    if (wg == 1) return launch_nt<F16, float, 1>(a, nt, grid, smem, st);
    if (wg == 2) return launch_nt<F16, float, 2>(a, nt, grid, smem, st);
    return launch_nt<F16, float, 4>(a, nt, grid, smem, st);
}

// How the rows are shared out: up to 64 columns a row block, an f32 row being three.
struct Shape {
    int blocks, block_rows, nt;
    Shape(int rows, int dtype) {
        const int split = dtype == TRBA_F32 ? 3 : 1, most = 64 / split;
        blocks = (rows + most - 1) / most;
        block_rows = (rows + blocks - 1) / blocks;
        nt = (block_rows * split + 7) / 8;
        if (nt == 7) nt = 8;
    }
    i64 workspace(int chunks) const { return nt > 1 ? (i64)blocks * chunks * 4 * nt * 512 : 0; }
};

int forward(const trba_linear_int4 *l, const void *x, int dtype, i64 ldx, int rows, void *y, i64 ldy, void *workspace,
            cudaStream_t st) {
    const Shape shape(rows, dtype);
    Args a{};
    a.cs = 1;
    a.blocks = l->base, a.bias = l->bias;
    a.x = x, a.y = y, a.ldx = ldx, a.ldy = ldy;
    a.frags = static_cast<uint4 *>(workspace);
    a.in = l->in, a.out = l->out, a.rows = rows, a.dtype = dtype;
    a.tiles = l->tiles, a.chunks = l->chunks;
    const bool scale_f16 = l->scale_dtype == TRBA_F16;
    const int nt = shape.nt, blocks_y = shape.blocks;
    a.block_rows = shape.block_rows;
    i64 smem = 0;
    int ctas = 0;
    if (nt > 1) {
        int4_fragments_kernel<<<dim3(grid_for((i64)l->chunks * 16 * a.block_rows), blocks_y), 256, 0, st>>>(a, nt);
        if (const int e = launched()) return e;
        // Tiles side by side: the fewest steps of the CTA with the most.
        i64 best = -1;
        for (int wn = kManyWarps; wn >= 1; wn >>= 1) {
            const int wk = kManyWarps / wn, red = wn * (wk - 1) * nt * 512;
            const int ks = many_blocks(nt);
            const i64 stages = (i64)many_depth(nt) * ks * (wk * nt * 2048 + kManyWarps * l->block);
            if (stages + red > kMaxSmem) break;
            const int groups = (a.tiles + wn - 1) / wn, grid = groups < sm_count() ? groups : sm_count();
            // A split over clusters leaves every CTA one group.  Clusters of 8
            // do not all find 8 free SMs next to each other on a full device:
            // 16 of them ran 24.5 us where 32 of 4 ran 16.4.
            int cs = 1;
            const auto fits = [&](int c) { return c * groups <= (c == 8 ? 96 : c == 4 ? 128 : sm_count()); };
            while (cs < 8 && fits(2 * cs) && 2 * cs * wk * ks <= a.chunks) cs *= 2;
            const i64 each = (a.chunks + cs - 1) / cs;
            const i64 cost = (i64)((groups + grid - 1) / grid) * ((each + wk * ks - 1) / (wk * ks) * ks + 1) + (cs > 1 ? 2 : 0);
            if (best < 0 || cost <= best)
                best = cost, a.wn = wn, a.cs = cs, ctas = grid * cs, a.red_at = (int)stages, smem = stages + red;
        }
    } else {
        const int cols = rows * (dtype == TRBA_F32 ? 3 : 1);
        const int ring = kFewWarps * kFewStages * kPair * l->block;
        const auto x_bytes = [&](int chunks) { return (cols * ((i64)chunks * 256 + 64) + 127) & ~127ll; };
        for (ctas = a.tiles < sm_count() ? a.tiles : sm_count();; ctas = ctas * 2 < a.tiles ? ctas * 2 : a.tiles) {
            const int share = (a.tiles + ctas - 1) / ctas;  // tiles of a CTA, at most
            // Tiles of a CTA that run side by side: the fewest steps of (chunks a
            // warp streams + the join of the warps that share a tile).
            i64 best = -1;
            int red = 0;
            for (int wn = kFewWarps; wn >= 1; wn >>= 1) {
                const int wk = kFewWarps / wn, bytes = 2 * wn * (wk - 1) * 512;
                const i64 steps = (share + wn - 1) / wn;
                const i64 cost = steps * (4 * ((a.chunks + wk - 1) / wk) + (wk > 1 ? 4 + wk : 0));
                if (best < 0 || cost < best) best = cost, a.wn = wn, red = bytes;
            }
            // All activations at once where they fit; else as many chunks as fit
            // beside the sums that wait between slabs.  Sums that leave no room
            // for a slab of a few chunks go to more CTAs.
            const i64 room = kMaxSmem - ring - red;
            i64 sums = 0;
            a.slab = a.chunks;
            if (x_bytes(a.chunks) > room) {
                sums = (i64)share * 512;
                a.slab = (int)(((room - sums - 128) / cols - 64) / 256);
                if (a.slab < 4 && ctas < a.tiles) continue;
            }
            a.xs_at = ring;
            a.red_at = a.xs_at + (int)x_bytes(a.slab);
            a.sums_at = a.red_at + red;
            smem = a.sums_at + sums;
            break;
        }
    }
    TRBA_REQUIRE_RET(smem > 0 && smem <= kMaxSmem, "trba_linear_int4_forward: shared memory", -1);
    const int wg = l->group >= 128 ? 4 : l->group / 32;
    const dim3 grid(ctas, blocks_y);
    return dtype == TRBA_F16 ? launch_type<true>(a, scale_f16, wg, nt, grid, smem, st)
                             : launch_type<false>(a, scale_f16, wg, nt, grid, smem, st);
}

template <class S>
int layout(trba_linear_int4 *l, const uint8_t *codes, i64 pitch, const void *scales, i64 ld_scales, cudaStream_t st) {
    int4_layout_kernel<S><<<grid_for((i64)l->tiles * l->chunks * 32), 256, 0, st>>>(
        codes, pitch, static_cast<const S *>(scales), ld_scales, l->in, l->out, l->group, l->groups, l->gpc, l->tiles,
        l->chunks, l->block, l->base);
    return launched();
}

bool sizes_ok(int in, int out, int group) {
    return in > 0 && in <= (1 << 30) && out > 0 && out <= (1 << 30) && (group == 32 || group == 64 || (group >= 128 && group % 128 == 0));
}

void lay_out(trba_linear_int4 *l, int in, int out, int group, int scale_dtype) {
    l->in = in, l->out = out, l->group = group, l->groups = (in - 1) / group + 1;
    l->scale_dtype = scale_dtype;
    l->tiles = (out - 1) / 16 + 1;
    l->chunks = (in - 1) / 128 + 1;
    l->gpc = group >= 128 ? 1 : 128 / group;
    l->block = 1024 + 16 * l->gpc * (scale_dtype == TRBA_F32 ? 4 : 2);
}
size_t blocks_bytes(const trba_linear_int4 *l) { return (size_t)l->tiles * l->chunks * l->block; }

trba_linear_int4 *allocate(int in, int out, int group, int scale_dtype, void *storage) {
    auto *l = new (std::nothrow) trba_linear_int4;
    if (!l) return nullptr;
    lay_out(l, in, out, group, scale_dtype);
    l->owned = !storage;
    l->base = static_cast<uint8_t *>(storage);
    if (cudaGetDevice(&l->device) != cudaSuccess ||
        (l->owned && cudaMalloc(&l->base, blocks_bytes(l) + (size_t)out * 4) != cudaSuccess)) {
        cudaGetLastError();
        report_error(__FILE__, __LINE__, "LinearInt4: device allocation failed", -1);
        delete l;
        return nullptr;
    }
    l->bias = reinterpret_cast<float *>(l->base + blocks_bytes(l));
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
    trba_linear_int4 *l = allocate(in_features, out_features, group, TRBA_F32, nullptr);
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

long long trba_linear_int4_bytes(int in_features, int out_features, int group, int scale_dtype) {
    if (!sizes_ok(in_features, out_features, group) || (scale_dtype != TRBA_F32 && scale_dtype != TRBA_F16)) return -1;
    trba_linear_int4 l;
    lay_out(&l, in_features, out_features, group, scale_dtype);
    return (long long)(blocks_bytes(&l) + (size_t)out_features * 4);
}

trba_linear_int4 *trba_linear_int4_create_codes(int in_features, int out_features, int group, const uint8_t *codes,
                                                long long ld_codes, const void *scales, int scale_dtype,
                                                long long ld_scales, const float *bias, void *storage,
                                                long long storage_bytes, void *stream) {
    TRBA_REQUIRE_RET(sizes_ok(in_features, out_features, group) && codes && scales &&
                         (scale_dtype == TRBA_F32 || scale_dtype == TRBA_F16) && ld_codes >= (in_features + 1ll) / 2 &&
                         ld_scales >= (in_features - 1) / group + 1,
                     "trba_linear_int4_create_codes: bad arguments", nullptr);
    TRBA_REQUIRE_RET(!storage || (storage_bytes >= trba_linear_int4_bytes(in_features, out_features, group, scale_dtype) &&
                                  reinterpret_cast<uintptr_t>(storage) % 16 == 0),
                     "trba_linear_int4_create_codes: storage too small or not aligned to 16 bytes", nullptr);
    trba_linear_int4 *l = allocate(in_features, out_features, group, scale_dtype, storage);
    if (!l) return nullptr;
    cudaStream_t st = as_stream(stream);
    bool ok = (scale_dtype == TRBA_F16 ? layout<__half>(l, codes, ld_codes, scales, ld_scales, st)
                                       : layout<float>(l, codes, ld_codes, scales, ld_scales, st)) == 0;
    ok = ok && (bias ? cudaMemcpyAsync(l->bias, bias, (size_t)out_features * 4, cudaMemcpyDeviceToDevice, st)
                     : cudaMemsetAsync(l->bias, 0, (size_t)out_features * 4, st)) == cudaSuccess;
    if (!storage && cudaStreamSynchronize(st) != cudaSuccess) ok = false;
    if (!ok) {
        report_error(__FILE__, __LINE__, "trba_linear_int4_create_codes: copying the weights failed", -1);
        trba_linear_int4_destroy(l);
        return nullptr;
    }
    return l;
}

void trba_linear_int4_destroy(trba_linear_int4 *l) {
    if (!l) return;
    if (l->owned) cudaFree(l->base);
    delete l;
}

long long trba_linear_int4_workspace(const trba_linear_int4 *l, int dtype, int rows) {
    return l && rows > 0 ? Shape(rows, dtype).workspace(l->chunks) : 0;
}

int trba_linear_int4_forward(const trba_linear_int4 *l, const void *x, int dtype, long long ldx, int rows, void *y,
                             long long ldy, void *workspace, long long workspace_bytes, void *stream) {
    TRBA_REQUIRE_RET(l && rows >= 0 && rows <= 1000000, "trba_linear_int4_forward: bad arguments", -1);
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
    const long long need = trba_linear_int4_workspace(l, dtype, rows);
    TRBA_REQUIRE_RET(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                     "trba_linear_int4_forward: workspace missing, too small or not aligned to 16 bytes", -1);
    return forward(l, x, dtype, ldx, rows, y, ldy, workspace, as_stream(stream));
}

int trba_linear_int4_get(const trba_linear_int4 *l, uint8_t *codes, float *scales, float *bias) {
    if (!l) return -1;
    int dev = -1;
    cudaGetDevice(&dev);
    TRBA_REQUIRE_RET(dev == l->device, "trba_linear_int4_get: the layer is on another device", -1);
    cudaError_t e = cudaDeviceSynchronize();
    if (codes && e == cudaSuccess) {
        const size_t n = (size_t)l->out * (((size_t)l->in + 1) / 2);
        uint8_t *nat = nullptr;
        e = cudaMalloc(&nat, n);
        if (e == cudaSuccess) {
            int4_natural_kernel<<<grid_for((i64)n), 256>>>(l->base, l->in, l->out, l->chunks, l->block, nat);
            e = (cudaError_t)launched();
            if (e == cudaSuccess) e = cudaMemcpy(codes, nat, n, cudaMemcpyDeviceToHost);
            cudaFree(nat);
        }
    }
    if (bias && e == cudaSuccess) e = cudaMemcpy(bias, l->bias, (size_t)l->out * 4, cudaMemcpyDeviceToHost);
    if (scales && e == cudaSuccess) {
        const bool f16 = l->scale_dtype == TRBA_F16;
        const size_t sb = l->block - 1024, nb = (size_t)l->tiles * l->chunks;  // the blocks' scales alone
        uint8_t *tmp = new (std::nothrow) uint8_t[nb * sb];
        TRBA_REQUIRE_RET(tmp, "trba_linear_int4_get: out of host memory", -1);
        e = cudaMemcpy2D(tmp, sb, l->base + 1024, l->block, sb, nb, cudaMemcpyDeviceToHost);
        for (int n = 0; n < l->out; ++n)
            for (int g = 0; g < l->groups; ++g) {
                const size_t chunk = (size_t)g * l->group / 128, part = l->group < 128 ? g % l->gpc : 0;
                const uint8_t *p = tmp + ((size_t)(n >> 4) * l->chunks + chunk) * sb;
                const size_t at = part * 16 + (n & 15);
                scales[(size_t)n * l->groups + g] = f16 ? __half2float(reinterpret_cast<const __half *>(p)[at])
                                                        : reinterpret_cast<const float *>(p)[at];
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
