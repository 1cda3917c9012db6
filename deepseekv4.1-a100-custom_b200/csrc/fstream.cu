// The products of decode-sized batches (up to 16 rows of x), bf16 / fp16 or FP8: every weight is used once per 8 rows, so the weight stream from
// HBM is the time, and what matters is that loads are in flight all the time.
//
// A block owns a tile of 16 weight rows (gated product: 8 gate rows and the 8 up rows that belong to them); its 8 warps split k.  The weights are
// the 16-row operand of mma.sync, 8 rows of x the other one; both go straight from global memory into the fragments, 16 bytes per thread: a
// thread's consecutive k of a row serve as the k words of an instruction in the same order for both operands, which a sum over k does not notice.
// x is read at its use: after the first tile of an SM it is in L1, which the weights bypass.  The warps' partial sums meet in shared memory in warp
// order (the same result from run to run).  The legacy mma.sync is enough here: at full HBM rate an SM issues one per 11 ns.
//
// Measured (graph replay, weights from HBM, with bias and residual): 1 x 4096 x 2048 5.2 us, 8 x 4096 x 4096 9.1, 8 x 12288 x 4096 20.0 (5.0 TB/s); FP8
// 8 x 4096 x 4096 7.3, 8 x 12288 x 4096 17.1.  What bounds it: a block's life (load, multiply, add up, store) is about 5 us of latencies, and an SM holds two or three;
// blocks that walk several tiles with the next loads in flight were slower (22.1 and 17.1 us for the 12288 rows: fewer warps fit).
#include "fgemm.cuh"

#include "common.cuh"
#include "ftypes.cuh"

namespace b200 {

constexpr int FS_WARPS = 8;

struct FsArgs {
    FgArgs g;
    int steps;  // of a warp along its share of k
    // FP8 form
    const uint8_t *xsf, *s8;
    int s_cols;
};

// This thread's place: weight rows lo / hi of a tile (gr and gr + 8), quarter t of a row's 64 bytes
struct FsLane { int warp, gr, t; };

__device__ __forceinline__ void mma_16816(__nv_bfloat16, float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
}
__device__ __forceinline__ void mma_16816(__half, float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 values at k of a row of K values, zeros behind its end (K need not be a multiple of 8; what follows it in memory is not read)
template <bool STREAM>
__device__ __forceinline__ uint4 load_k8(const uint16_t* row, int k, int K) {
    if (k + 8 <= K) return STREAM ? ldg_stream16(row + k) : __ldg(reinterpret_cast<const uint4*>(row + k));
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k + i < K) v[i >> 1] |= (uint32_t)row[k + i] << (16 * (i & 1));
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// ------------------------------------------------------------------ 16-bit operands: a step is U groups of 32 k
template <typename T_, int NT, int U>
struct FsHalf {
    using T = T_;
    struct Buf { uint4 lo[U], hi[U]; };
    const uint16_t *w, *x[NT];
    bool x_on[NT];
    int g_lo, g_hi, K;

    static __host__ __device__ int steps(int K) { return ((K + 31) / 32 + FS_WARPS * U - 1) / (FS_WARPS * U); }

    __device__ FsHalf(const FsArgs& a, const FsLane& l) {
        const FgArgs& g = a.g;
        const int groups = (g.K + 31) / 32;
        g_lo = (int)((long long)groups * l.warp / FS_WARPS);
        g_hi = (int)((long long)groups * (l.warp + 1) / FS_WARPS);
        K = g.K - l.t * 8;
        w = reinterpret_cast<const uint16_t*>(g.b.base) + l.t * 8;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            x_on[j] = j * 8 + l.gr < g.M;
            x[j] = reinterpret_cast<const uint16_t*>(g.a.base) + (long long)(x_on[j] ? j * 8 + l.gr : 0) * g.a.ld + l.t * 8;
        }
    }
    __device__ __forceinline__ void load(const FsArgs& a, int row_lo, bool on_lo, int row_hi, bool on_hi, int step, Buf& b) const {
        const uint16_t *p = w + (long long)(on_lo ? row_lo : 0) * a.g.b.ld, *q = w + (long long)(on_hi ? row_hi : 0) * a.g.b.ld;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int gi = g_lo + step * U + i;
            const bool in = gi < g_hi;
            b.lo[i] = in && on_lo ? load_k8<true>(p, gi * 32, K) : make_uint4(0, 0, 0, 0);
            b.hi[i] = in && on_hi ? load_k8<true>(q, gi * 32, K) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void multiply(int step, const Buf& b, float (&acc)[NT][4]) const {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            uint4 v[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int gi = g_lo + step * U + i;
                v[i] = gi < g_hi && x_on[j] ? load_k8<false>(x[j], gi * 32, K) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                mma_16816(T(), acc[j], b.lo[i].x, b.hi[i].x, b.lo[i].y, b.hi[i].y, v[i].x, v[i].y);
                mma_16816(T(), acc[j], b.lo[i].z, b.hi[i].z, b.lo[i].w, b.hi[i].w, v[i].z, v[i].w);
            }
        }
    }
};

// ------------------------------------------------------------------ FP8 operands: a step is U units of 128 k
// e4m3 weights with one E8M0 scale per 32 rows x 32 k, e4m3 rows of x with one per 32 k: mma.sync.m16n8k32 takes the codes as they are; a
// thread's 8 bytes of a 32-k group are the two k words of one instruction.  Each group's product starts from zero and is added times the group's
// two scales, which are the same for all 16 weight rows of the tile.  The four threads of a row load 64 bytes, 16 each, which leaves group 0 with
// threads 0, 1 and group 1 with threads 2, 3; threads t and t ^ 2 then swap halves, so that each has 8 bytes of both groups.
__device__ __forceinline__ void mma_e4m3_16832(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// v: 16 bytes of this thread; afterwards (x, y): its 8 bytes of group 0, (z, w): its 8 bytes of group 1
__device__ __forceinline__ uint4 swap_groups(uint4 v, bool upper) {
    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, upper ? v.x : v.z, 2), r1 = __shfl_xor_sync(0xffffffffu, upper ? v.y : v.w, 2);
    return upper ? make_uint4(r0, r1, v.z, v.w) : make_uint4(v.x, v.y, r0, r1);
}
__device__ __forceinline__ float e8m0_f32(uint32_t b) { return u32_as_f32(b ? b << 23 : 0x00400000u); }  // 2^(b - 127)

template <int NT, int U>
struct FsQ8 {
    using T = __nv_bfloat16;
    struct Buf { uint4 lo[U * 2], hi[U * 2]; uint32_t ws[U]; };
    const uint8_t *w, *x[NT];
    const uint32_t *sx0[NT], *sx1[NT];
    bool x_on[NT], upper;
    int u_lo, u_hi;

    static __host__ __device__ int steps(int K) { return (K / 128 + FS_WARPS * U - 1) / (FS_WARPS * U); }

    __device__ FsQ8(const FsArgs& a, const FsLane& l) {
        const FgArgs& g = a.g;
        const int units = g.K / 128, sx_ld = g.K / 128;
        u_lo = (int)((long long)units * l.warp / FS_WARPS);
        u_hi = (int)((long long)units * (l.warp + 1) / FS_WARPS);
        upper = l.t >= 2;
        w = reinterpret_cast<const uint8_t*>(g.b.base) + l.t * 16;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            x_on[j] = j * 8 + l.gr < g.M;
            // the bytes of a group that this thread has after the swap: 0, 16, 8, 24 for t = 0 .. 3
            x[j] = reinterpret_cast<const uint8_t*>(g.a.base) + (long long)(x_on[j] ? j * 8 + l.gr : 0) * g.K + (l.t & 1) * 16 + (l.t >> 1) * 8;
            const int m0 = j * 8 + 2 * l.t;  // the rows of x of this thread's accumulators; rows behind the last one borrow its scales
            sx0[j] = reinterpret_cast<const uint32_t*>(a.xsf) + (long long)min(m0, g.M - 1) * sx_ld;
            sx1[j] = reinterpret_cast<const uint32_t*>(a.xsf) + (long long)min(m0 + 1, g.M - 1) * sx_ld;
        }
    }
    __device__ __forceinline__ void load(const FsArgs& a, int row_lo, bool on_lo, int row_hi, bool on_hi, int step, Buf& b) const {
        const uint8_t *p = w + (long long)(on_lo ? row_lo : 0) * a.g.K, *q = w + (long long)(on_hi ? row_hi : 0) * a.g.K;
        const uint8_t* s = a.s8 + (long long)((on_lo ? row_lo : 0) >> 5) * a.s_cols;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = u_lo + step * U + i;
            const bool in = u < u_hi;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                b.lo[2 * i + h] = in && on_lo ? ldg_stream16(p + u * 128 + h * 64) : make_uint4(0, 0, 0, 0);
                b.hi[2 * i + h] = in && on_hi ? ldg_stream16(q + u * 128 + h * 64) : make_uint4(0, 0, 0, 0);
            }
            b.ws[i] = in ? __ldg(s + u * 4) | __ldg(s + u * 4 + 1) << 8 | __ldg(s + u * 4 + 2) << 16 | (uint32_t)__ldg(s + u * 4 + 3) << 24 : 0;
        }
    }
    __device__ __forceinline__ void multiply(int step, const Buf& b, float (&acc)[NT][4]) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = u_lo + step * U + i;
            const bool in = u < u_hi;
            uint4 lo[2], hi[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) { lo[h] = swap_groups(b.lo[2 * i + h], upper); hi[h] = swap_groups(b.hi[2 * i + h], upper); }
            uint32_t ws = b.ws[i];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                uint2 v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = in && x_on[j] ? __ldg(reinterpret_cast<const uint2*>(x[j] + u * 128 + q * 32)) : make_uint2(0, 0);
                const uint32_t s0 = in ? __ldg(sx0[j] + u) : 0, s1 = in ? __ldg(sx1[j] + u) : 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float p[4];
                    if (q & 1) mma_e4m3_16832(p, lo[q >> 1].z, hi[q >> 1].z, lo[q >> 1].w, hi[q >> 1].w, v[q].x, v[q].y);
                    else mma_e4m3_16832(p, lo[q >> 1].x, hi[q >> 1].x, lo[q >> 1].y, hi[q >> 1].y, v[q].x, v[q].y);
                    const float f = e8m0_f32((ws >> (8 * q)) & 0xFFu), f0 = f * e8m0_f32((s0 >> (8 * q)) & 0xFFu), f1 = f * e8m0_f32((s1 >> (8 * q)) & 0xFFu);
                    acc[j][0] = fmaf(p[0], f0, acc[j][0]);
                    acc[j][1] = fmaf(p[1], f1, acc[j][1]);
                    acc[j][2] = fmaf(p[2], f0, acc[j][2]);
                    acc[j][3] = fmaf(p[3], f1, acc[j][3]);
                }
            }
        }
    }
};

// ------------------------------------------------------------------ the kernel
template <typename Op, int NT, bool DUAL, int BLOCKS>
__global__ void __launch_bounds__(FS_WARPS * 32, BLOCKS) fs_kernel(const FsArgs a) {
    using T = typename Op::T;
    __shared__ float part[FS_WARPS][NT * 8][17];
    pdl_wait();
    pdl_launch_dependents();
    const FgArgs& g = a.g;
    const int lane = threadIdx.x & 31;
    const FsLane l{(int)threadIdx.x >> 5, lane >> 2, lane & 3};
    constexpr int COLS = DUAL ? 8 : 16;
    const int width = DUAL ? g.inter : g.N, col0 = blockIdx.x * COLS;
    const int row_lo = col0 + l.gr, row_hi = DUAL ? g.inter + row_lo : row_lo + 8;
    const bool on_lo = row_lo < width, on_hi = DUAL ? on_lo : row_hi < width;
    const Op op(a, l);
    float acc[NT][4] = {};
    for (int step = 0; step < a.steps; ++step) {
        typename Op::Buf b;
        op.load(a, row_lo, on_lo, row_hi, on_hi, step, b);
        op.multiply(step, b, acc);
    }
    // acc[j] = rows gr, gr, gr + 8, gr + 8 of the tile against rows 2 t, 2 t + 1, 2 t, 2 t + 1 of x (+ 8 j)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        float(*p)[17] = part[l.warp];
        p[j * 8 + 2 * l.t][l.gr] = acc[j][0];
        p[j * 8 + 2 * l.t + 1][l.gr] = acc[j][1];
        p[j * 8 + 2 * l.t][l.gr + 8] = acc[j][2];
        p[j * 8 + 2 * l.t + 1][l.gr + 8] = acc[j][3];
    }
    const int m = threadIdx.x / COLS, c = threadIdx.x - m * COLS, col = col0 + c;  // NT * 8 * COLS <= the block's threads
    const bool mine = m < NT * 8 && m < g.M && col < width;
    float bias = 0.f, res = 0.f;
    if (!DUAL && mine) {
        if (g.bias) bias = to_f32(reinterpret_cast<const T*>(g.bias)[col]);
        if (g.res) res = to_f32(reinterpret_cast<const T*>(g.res)[m * g.res_ld + col]);
    }
    __syncthreads();
    if (!mine) return;
    float z = 0.f;
#pragma unroll
    for (int w = 0; w < FS_WARPS; ++w) z += part[w][m][c];
    if constexpr (DUAL) {
        float u = 0.f;
#pragma unroll
        for (int w = 0; w < FS_WARPS; ++w) u += part[w][m][c + 8];
        if (g.z_out) {
            g.z_out[m * g.z_ld + col] = z;
            g.z_out[m * g.z_ld + g.inter + col] = u;
        }
        if (g.limit > 0.f) {
            z = z > g.limit ? g.limit : z;
            u = u > g.limit ? g.limit : (u < -g.limit ? -g.limit : u);
        }
        z = act_fwd(g.act, z) * u;
    } else {
        z += bias;
        if (g.z_out) g.z_out[m * g.z_ld + col] = z;
        z = act_fwd(g.act, z) + res;
    }
    reinterpret_cast<T*>(g.out)[m * g.out_ld + col] = from_f32<T>(z);
}

int sm_count();

template <typename Op, int NT, bool DUAL, int BLOCKS>
static int fs_run(FsArgs& a, int tiles, cudaStream_t stream) {
    a.steps = Op::steps(a.g.K);
    return (int)launch_pdl(fs_kernel<Op, NT, DUAL, BLOCKS>, dim3(tiles), dim3(FS_WARPS * 32), 0, stream, a);
}

static int fs_tiles(const FgArgs& g) { return g.dual ? (g.inter + 7) / 8 : (g.N + 15) / 16; }

// All blocks resident at once: long steps (8 x 4096 x 4096: 8.5 us with 8 groups in flight, 9.7 with 4); more blocks than that: shorter steps and three
// blocks per SM (8 x 12288 x 4096: 19.1 us against 21.6; 16 rows: 25.2 against 28.6).
template <typename T, int NT, bool DUAL>
static int fs_half(FsArgs& a, cudaStream_t stream) {
    const int tiles = fs_tiles(a.g);
    if (tiles <= 2 * sm_count()) return fs_run<FsHalf<T, NT, 8>, NT, DUAL, 2>(a, tiles, stream);
    return fs_run<FsHalf<T, NT, 4>, NT, DUAL, 3>(a, tiles, stream);
}

template <typename T>
static int fs_typed(FsArgs& a, cudaStream_t stream) {
    if (a.g.M <= 8) return a.g.dual ? fs_half<T, 1, true>(a, stream) : fs_half<T, 1, false>(a, stream);
    return a.g.dual ? fs_half<T, 2, true>(a, stream) : fs_half<T, 2, false>(a, stream);
}

int fs_launch(const FgArgs& g, cudaStream_t stream) {
    FsArgs a{};
    a.g = g;
    return g.is_f16 ? fs_typed<__half>(a, stream) : fs_typed<__nv_bfloat16>(a, stream);
}

int fs_q8_launch(const FgArgs& g, const uint8_t* xsf, const uint8_t* s8, int s_cols, cudaStream_t stream) {
    FsArgs a{};
    a.g = g;
    a.xsf = xsf;
    a.s8 = s8;
    a.s_cols = s_cols;
    const int tiles = fs_tiles(g);
    // 8 x 4096 x 4096: 7.2 us with two blocks per SM, 8.6 with three (fewer registers for loads); 8 x 12288 x 4096: 17.6 against 15.9
    if (g.M > 8) return fs_run<FsQ8<2, 2>, 2, false, 2>(a, tiles, stream);
    if (tiles <= 2 * sm_count()) return fs_run<FsQ8<1, 2>, 1, false, 2>(a, tiles, stream);
    return fs_run<FsQ8<1, 2>, 1, false, 3>(a, tiles, stream);
}

}  // namespace b200
