// The 16-bit products of decode-sized batches (up to 16 rows of x): every weight is used once per 8 rows, so the weight stream from HBM is the
// time, and what matters is how many bytes are in flight.
//
// A block owns 16 weight rows (gated product: 8 gate rows and the 8 up rows that belong to them) and its 8 warps split k.  The weights are the
// 16-row operand of mma.sync.m16n8k16, 8 rows of x the other one; both go straight from global memory into the fragments, 16 bytes per
// thread: a thread's 8 consecutive k of a row serve as the k pairs of two instructions, in the same order for both operands, which a sum over k
// does not notice.  No shared memory before the end, where the warps' partial sums are added in warp order (the same result from run to run).
// The legacy mma.sync is enough here: at full HBM rate an SM issues one per 11 ns.
#include "fgemm.cuh"

#include "common.cuh"
#include "ftypes.cuh"

namespace b200 {

constexpr int FS_WARPS = 8;
constexpr int FS_UNROLL = 4;  // groups of 32 k in flight per warp and row half

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

template <typename T, int NT, bool DUAL>
__global__ void __launch_bounds__(FS_WARPS * 32) fs_kernel(const FgArgs g) {
    __shared__ float part[FS_WARPS][NT * 8][17];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
    const int n_cols = DUAL ? 8 : 16, col0 = blockIdx.x * n_cols, width = DUAL ? g.inter : g.N;
    // the two weight rows of this thread: gr and gr + 8 of the tile
    const int c_lo = col0 + gr, c_hi = DUAL ? g.inter + c_lo : c_lo + 8;
    const bool on_lo = c_lo < width, on_hi = DUAL ? on_lo : c_hi < width;
    const uint16_t* w_lo = reinterpret_cast<const uint16_t*>(g.b.base) + (long long)(on_lo ? c_lo : 0) * g.b.ld + t * 8;
    const uint16_t* w_hi = reinterpret_cast<const uint16_t*>(g.b.base) + (long long)(on_hi ? c_hi : 0) * g.b.ld + t * 8;
    const uint16_t* xr[NT];
    bool x_on[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        x_on[j] = j * 8 + gr < g.M;
        xr[j] = reinterpret_cast<const uint16_t*>(g.a.base) + (long long)(x_on[j] ? j * 8 + gr : 0) * g.a.ld + t * 8;
    }
    const int groups = (g.K + 31) / 32, g_end = (int)((long long)groups * (warp + 1) / FS_WARPS), K = g.K - t * 8;
    float acc[NT][4] = {};
    for (int q = (int)((long long)groups * warp / FS_WARPS); q < g_end; q += FS_UNROLL) {
        uint4 lo[FS_UNROLL], hi[FS_UNROLL], xv[FS_UNROLL][NT];
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < FS_UNROLL; ++i) {
            const int k = (q + i) * 32;
            const bool in = q + i < g_end;
            lo[i] = in && on_lo ? load_k8<true>(w_lo, k, K) : zero;
            hi[i] = in && on_hi ? load_k8<true>(w_hi, k, K) : zero;
#pragma unroll
            for (int j = 0; j < NT; ++j) xv[i][j] = in && x_on[j] ? load_k8<false>(xr[j], k, K) : zero;
        }
#pragma unroll
        for (int i = 0; i < FS_UNROLL; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                mma_16816(T(), acc[j], lo[i].x, hi[i].x, lo[i].y, hi[i].y, xv[i][j].x, xv[i][j].y);
                mma_16816(T(), acc[j], lo[i].z, hi[i].z, lo[i].w, hi[i].w, xv[i][j].z, xv[i][j].w);
            }
    }
    // acc[j] = rows gr, gr, gr + 8, gr + 8 of the tile against rows 2 t, 2 t + 1, 2 t, 2 t + 1 of x (+ 8 j)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        part[warp][j * 8 + 2 * t][gr] = acc[j][0];
        part[warp][j * 8 + 2 * t + 1][gr] = acc[j][1];
        part[warp][j * 8 + 2 * t][gr + 8] = acc[j][2];
        part[warp][j * 8 + 2 * t + 1][gr + 8] = acc[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * n_cols; i += FS_WARPS * 32) {
        const int m = i / n_cols, c = i - m * n_cols, col = col0 + c;
        if (m >= g.M || col >= width) continue;
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
            if (g.bias) z += to_f32(reinterpret_cast<const T*>(g.bias)[col]);
            if (g.z_out) g.z_out[m * g.z_ld + col] = z;
            z = act_fwd(g.act, z);
            if (g.res) z += to_f32(reinterpret_cast<const T*>(g.res)[m * g.res_ld + col]);
        }
        reinterpret_cast<T*>(g.out)[m * g.out_ld + col] = from_f32<T>(z);
    }
}

template <typename T, int NT>
static int fs_run(const FgArgs& a, cudaStream_t stream) {
    const int cols = a.dual ? 8 : 16, width = a.dual ? a.inter : a.N;
    return (int)launch_pdl(a.dual ? fs_kernel<T, NT, true> : fs_kernel<T, NT, false>, dim3((width + cols - 1) / cols), dim3(FS_WARPS * 32), 0, stream, a);
}

int fs_launch(const FgArgs& a, cudaStream_t stream) {
    if (a.M <= 8) return a.is_f16 ? fs_run<__half, 1>(a, stream) : fs_run<__nv_bfloat16, 1>(a, stream);
    return a.is_f16 ? fs_run<__half, 2>(a, stream) : fs_run<__nv_bfloat16, 2>(a, stream);
}

}  // namespace b200
