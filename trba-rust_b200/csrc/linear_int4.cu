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

namespace cg = cooperative_groups;

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
// y^T = W x^T on the tensor cores: A is a 16-output tile of the weights, the
// codes turned into exact bf16 or f16 integers in registers, B the
// activations from shared memory, eight columns at a time.  An f32
// activation enters as three bf16 columns whose sum it is exactly, so its
// products with the codes are exact in all types, and a group's sum is
// accumulated in f32 before its scale multiplies it.
//
// What bounds it: at one row, reading the codes (half a byte a weight).  The
// legacy mma is enough for that: a 1 KB block of codes costs 8 mma per eight
// columns and about 90 integer and conversion instructions.
//
// A CTA is 8 warps, wn tiles by wk interleaved parts of its inputs; a
// cluster of `cs` CTAs splits the inputs once more and adds its parts through
// distributed shared memory, so there is no workspace and the order of every
// sum is fixed.  Each warp streams its blocks through its own ring of
// cp.async stages, which are in flight while the activations are staged.
constexpr int kWarps = 8, kDepth = 6;

struct Args {
    const uint8_t *codes, *scales;
    const float *bias;
    const void *x;
    void *y;
    i64 ldx, ldy;
    int in, out, rows, dtype;
    int tiles, chunks, group, gpc, groups_pad, scale_f16;
    int wn, cs;          // wk = kWarps / wn
    int slab;            // chunks whose activations are staged at once, a multiple of wk
    int block_rows;      // rows a CTA takes
    int cols;            // columns they make (3 a row for f32)
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// Eight activations of one row from k on (zero behind `in`) as 16-bit columns.
__device__ __forceinline__ void stage8(const Args &a, int row, int k, uint8_t *dst, int pitch) {
    if (a.dtype != TRBA_F32) {
        const uint16_t *src = static_cast<const uint16_t *>(a.x) + row * a.ldx + k;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k + 8 <= a.in && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            v = *reinterpret_cast<const uint4 *>(src);
        } else {
            uint16_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = k + i < a.in ? src[i] : (uint16_t)0;
            v.x = h[0] | (uint32_t)h[1] << 16, v.y = h[2] | (uint32_t)h[3] << 16;
            v.z = h[4] | (uint32_t)h[5] << 16, v.w = h[6] | (uint32_t)h[7] << 16;
        }
        *reinterpret_cast<uint4 *>(dst) = v;
        return;
    }
    const float *src = static_cast<const float *>(a.x) + row * a.ldx + k;
    float f[8];
    if (k + 8 <= a.in && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        const float4 lo = reinterpret_cast<const float4 *>(src)[0], hi = reinterpret_cast<const float4 *>(src)[1];
        f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = k + i < a.in ? src[i] : 0.0f;
    }
    uint32_t part[3][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // truncated to 8 bits three times: hi + mid + lo is the value; an
        // infinity or NaN goes in whole
        const bool finite = fabsf(f[i]) <= 3.402823466e38f;
        const uint32_t h = finite ? __float_as_uint(f[i]) & 0xffff0000u
                                  : (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(f[i])) << 16;
        const float r1 = finite ? f[i] - __uint_as_float(h) : 0.0f;
        const uint32_t m = __float_as_uint(r1) & 0xffff0000u;
        const uint32_t l = __float_as_uint(r1 - __uint_as_float(m)) & 0xffff0000u;
        const uint32_t q[3] = {h, m, l};
#pragma unroll
        for (int p = 0; p < 3; ++p) part[p][i >> 1] = i & 1 ? part[p][i >> 1] | q[p] : q[p] >> 16;
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
        *reinterpret_cast<uint4 *>(dst + (i64)p * pitch) = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
}

// WG: words (32 inputs) a group has in a chunk; NT: tiles of eight columns.
template <bool F16, int WG, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT <= 4 ? 2 : 1) int4_forward_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wk_n = kWarps / a.wn, wn = warp / wk_n, wk = warp - wn * wk_n;
    const int rank = blockIdx.x % a.cs, tile = (blockIdx.x / a.cs) * a.wn + wn;
    const int per = ((a.chunks + a.cs - 1) / a.cs + wk_n - 1) / wk_n * wk_n;  // chunks of a CTA
    const int c0 = rank * per, nc = max(0, min(a.chunks, c0 + per) - c0);
    const int row0 = blockIdx.y * a.block_rows, rows = min(a.block_rows, a.rows - row0);
    const int split = a.dtype == TRBA_F32 ? 3 : 1, cols = rows * split;
    const int es = a.scale_f16 ? 2 : 4, sb = 16 * a.gpc * es, slot = 1024 + sb;
    const int pitch = a.slab * 256 + 64;  // 64 mod 128: eight lanes' 16-byte reads meet 32 different banks
    uint8_t *ring = smem + warp * kDepth * slot;
    uint8_t *xs = smem + kWarps * kDepth * slot;
    const uint32_t ring_s = smem_addr(ring);
    const int mine = tile < a.tiles && wk < nc ? (nc - wk + wk_n - 1) / wk_n : 0;
    const uint8_t *src = a.codes + ((i64)tile * a.chunks + c0 + wk) * 1024;
    const uint8_t *ssrc = a.scales + (i64)tile * a.groups_pad * 16 * es;

    auto issue = [&](int i) {
        if (i < mine) {
            const uint32_t dst = ring_s + (i % kDepth) * slot;
            const uint8_t *p = src + (i64)i * wk_n * 1024;
            cp16(dst + lane * 16, p + lane * 16);
            cp16(dst + 512 + lane * 16, p + 512 + lane * 16);
            if (lane * 16 < sb) {
                const int chunk = c0 + wk + i * wk_n;
                const int g = WG < 4 ? chunk * (4 / WG) : (int)((i64)chunk * 128 / a.group);
                cp16(dst + 1024 + lane * 16, ssrc + (i64)g * 16 * es + lane * 16);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kDepth - 1; ++i) issue(i);

    float tot[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) tot[n][0] = tot[n][1] = tot[n][2] = tot[n][3] = 0.0f;
    const int g = lane >> 2, t = lane & 3;
    int i = 0;
    for (int s0 = 0; s0 < nc; s0 += a.slab) {
        const int sc = min(a.slab, nc - s0);
        if (s0) __syncthreads();
        for (int e = threadIdx.x; e < rows * sc * 16; e += kWarps * 32) {
            const int r = e / (sc * 16), k8 = e - r * sc * 16;
            stage8(a, row0 + r, (c0 + s0) * 128 + k8 * 8, xs + (i64)r * split * pitch + k8 * 16, pitch);
        }
        __syncthreads();
        for (; i < mine && wk + i * wk_n < s0 + sc; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
            __syncwarp();
            issue(i + kDepth - 1);
            const uint8_t *blk = ring + (i % kDepth) * slot;
            const uint4 lo = *reinterpret_cast<const uint4 *>(blk + lane * 16);
            const uint4 hi = *reinterpret_cast<const uint4 *>(blk + 512 + lane * 16);
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
            const uint8_t *xk = xs + (wk + i * wk_n - s0) * 256 + t * 16;
            float c[NT][4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (w % WG == 0) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
                }
                uint32_t a0[4], a1[4];
                a0[0] = code_pair<F16>(wl[w]), a0[1] = code_pair<F16>(wh[w]);
                a0[2] = code_pair<F16>(wl[w] >> 4), a0[3] = code_pair<F16>(wh[w] >> 4);
                a1[0] = code_pair<F16>(wl[w] >> 8), a1[1] = code_pair<F16>(wh[w] >> 8);
                a1[2] = code_pair<F16>(wl[w] >> 12), a1[3] = code_pair<F16>(wh[w] >> 12);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint4 b = make_uint4(0, 0, 0, 0);
                    if (n * 8 + g < cols) b = *reinterpret_cast<const uint4 *>(xk + (n * 8 + g) * pitch + w * 64);
                    mma<F16>(c[n], a0, b.x, b.y);
                    mma<F16>(c[n], a1, b.z, b.w);
                }
                if (w % WG == WG - 1) {
                    float s0f, s1f;
                    const uint8_t *sp = blk + 1024 + (w / WG) * 16 * es;
                    if (a.scale_f16) {
                        s0f = __half2float(reinterpret_cast<const __half *>(sp)[g]);
                        s1f = __half2float(reinterpret_cast<const __half *>(sp)[g + 8]);
                    } else {
                        s0f = reinterpret_cast<const float *>(sp)[g];
                        s1f = reinterpret_cast<const float *>(sp)[g + 8];
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        tot[n][0] = fmaf(s0f, c[n][0], tot[n][0]);
                        tot[n][1] = fmaf(s0f, c[n][1], tot[n][1]);
                        tot[n][2] = fmaf(s1f, c[n][2], tot[n][2]);
                        tot[n][3] = fmaf(s1f, c[n][3], tot[n][3]);
                    }
                }
            }
        }
    }
    // partial sums [wk][output][column] over the ring and the activations
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    constexpr int kCols = NT * 8 + 1;
    float *red = reinterpret_cast<float *>(smem);
    const int outs = a.wn * 16;
    {
        float *p = red + ((i64)wk * outs + wn * 16 + g) * kCols + 2 * t;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            p[n * 8] = tot[n][0], p[n * 8 + 1] = tot[n][1];
            p[8 * kCols + n * 8] = tot[n][2], p[8 * kCols + n * 8 + 1] = tot[n][3];
        }
    }
    __syncthreads();
    if (a.cs > 1) {
        for (int e = threadIdx.x; e < outs * kCols; e += kWarps * 32)
            for (int k = 1; k < wk_n; ++k) red[e] += red[(i64)k * outs * kCols + e];
        cg::this_cluster().sync();
    }
    const int n0 = (blockIdx.x / a.cs) * outs;
    for (int e = threadIdx.x + rank * kWarps * 32; e < rows * outs; e += kWarps * 32 * a.cs) {
        const int r = e / outs, o = e - r * outs;
        if (n0 + o >= a.out) continue;
        float v[3] = {0.0f, 0.0f, 0.0f};
        for (int p = 0; p < split; ++p) {
            const int at = o * kCols + r * split + p;
            if (a.cs > 1) {
                for (int k = 0; k < a.cs; ++k) v[p] += *cg::this_cluster().map_shared_rank(red + at, k);
            } else {
                for (int k = 0; k < wk_n; ++k) v[p] += red[(i64)k * outs * kCols + at];
            }
        }
        const float sum = v[0] + (v[1] + v[2]) + a.bias[n0 + o];
        const i64 at = (row0 + r) * a.ldy + n0 + o;
        if (a.dtype == TRBA_F32) static_cast<float *>(a.y)[at] = sum;
        else if (a.dtype == TRBA_BF16) static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(sum);
        else static_cast<__half *>(a.y)[at] = __float2half_rn(sum);
    }
    if (a.cs > 1) cg::this_cluster().sync();  // no CTA leaves while its sums are read
}

int launched() {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
    return (int)e;
}

constexpr int kMaxCols = 64;
constexpr int kSlabBytes = 48 * 1024;

template <bool F16, int WG, int NT>
int launch(const Args &a, int blocks_x, int blocks_y, size_t smem, cudaStream_t st) {
    auto fn = int4_forward_kernel<F16, WG, NT>;
    static std::atomic<unsigned long long> sized{0};  // one bit a device: its limit has been raised
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(sized.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(fn),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) {
            report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
            return (int)e;
        }
        sized.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = a.cs, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks_x, blocks_y);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, fn, a);
    return launched();
}

template <bool F16, int WG>
int launch_nt(const Args &a, int bx, int by, int cols, size_t smem, cudaStream_t st) {
    const int nt = (cols + 7) / 8;
    if (nt <= 1) return launch<F16, WG, 1>(a, bx, by, smem, st);
    if (nt <= 2) return launch<F16, WG, 2>(a, bx, by, smem, st);
    if (nt <= 4) return launch<F16, WG, 4>(a, bx, by, smem, st);
    return launch<F16, WG, 8>(a, bx, by, smem, st);
}

int forward(const trba_linear_int4 *l, const void *x, int dtype, i64 ldx, int rows, void *y, i64 ldy, cudaStream_t st) {
    Args a{};
    a.codes = l->codes, a.scales = l->scales, a.bias = l->bias;
    a.x = x, a.y = y, a.ldx = ldx, a.ldy = ldy;
    a.in = l->in, a.out = l->out, a.rows = rows, a.dtype = dtype;
    a.tiles = l->tiles, a.chunks = l->chunks, a.group = l->group, a.gpc = l->gpc;
    a.groups_pad = l->groups_pad, a.scale_f16 = l->scale_dtype == TRBA_F16;
    const int split = dtype == TRBA_F32 ? 3 : 1, most = kMaxCols / split;
    const int blocks_y = (rows + most - 1) / most;
    a.block_rows = (rows + blocks_y - 1) / blocks_y;
    a.cols = a.block_rows * split;
    const int target = 2 * sm_count();
    a.wn = kWarps;
    while (a.wn > 1 && (a.tiles + a.wn - 1) / a.wn * blocks_y < target) a.wn >>= 1;
    const int wk = kWarps / a.wn;
    const int blocks = (a.tiles + a.wn - 1) / a.wn;
    a.cs = 1;
    while (a.cs < 8 && blocks * blocks_y * a.cs < sm_count() && a.chunks >= 2 * a.cs * wk * 2) a.cs *= 2;
    const int per = ((a.chunks + a.cs - 1) / a.cs + wk - 1) / wk * wk;
    a.slab = (kSlabBytes / a.cols - 64) / 256 / wk * wk;
    if (a.slab < wk) a.slab = wk;
    if (a.slab > per) a.slab = per;
    const size_t slot = 1024 + 16 * a.gpc * (a.scale_f16 ? 2 : 4);
    const int nt = a.cols <= 8 ? 1 : a.cols <= 16 ? 2 : a.cols <= 32 ? 4 : 8;
    size_t smem = kWarps * kDepth * slot + (size_t)a.cols * (a.slab * 256 + 64);
    const size_t red = (size_t)kWarps * 16 * (nt * 8 + 1) * 4;
    if (smem < red) smem = red;
    const int wg = l->group >= 128 ? 4 : l->group / 32, bx = blocks * a.cs;
    if (dtype == TRBA_F16) {
        if (wg == 1) return launch_nt<true, 1>(a, bx, blocks_y, a.cols, smem, st);
        if (wg == 2) return launch_nt<true, 2>(a, bx, blocks_y, a.cols, smem, st);
        return launch_nt<true, 4>(a, bx, blocks_y, a.cols, smem, st);
    }
    if (wg == 1) return launch_nt<false, 1>(a, bx, blocks_y, a.cols, smem, st);
    if (wg == 2) return launch_nt<false, 2>(a, bx, blocks_y, a.cols, smem, st);
    return launch_nt<false, 4>(a, bx, blocks_y, a.cols, smem, st);
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
