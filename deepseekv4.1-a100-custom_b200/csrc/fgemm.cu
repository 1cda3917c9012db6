// 16-bit GEMM on the 5th-generation tensor cores (tcgen05.mma.kind::f16, TMA, TMEM) with the epilogues of the dense operators: bias,
// activation and residual, or the gated product of two projections.
//
// Persistent CTAs, one per SM, walk the output tiles; with CG = 2 a pair of SMs (a cluster of two CTAs) shares a tile of 256 x BN
// (tcgen05 cta_group::2): each SM fetches its own 128 rows of A and half of the rows of B, so a k block costs 16 + BN/16 KB of shared memory
// traffic per 128 x BN of results where a lone SM needs 16 + BN/8.  Warp roles:
//   warp 0      TMA producer: 64-deep k blocks of both operands into a ring of shared-memory stages (128-byte swizzle)
//   warp 1      one thread (of the first CTA of a pair) issues the MMAs; the accumulators live in TMEM, two buffers, so that the epilogue of
//               a tile runs under the MMAs of the next
//   warps 4-11  epilogue: a thread owns one output row (TMEM lane) and half of the tile's columns
// Every wait is bounded; one that runs out of time records a code in a device error word and the CTA runs to its end.
#include "fgemm.cuh"

#include "common.cuh"
#include "ftypes.cuh"
#include "tc5.cuh"

namespace b200 {

__device__ int g_fg_error = 0;

constexpr int FG_THREADS = 384;
constexpr int FG_BM = 128, FG_BK = 64;  // rows of A per CTA, depth of a k block
constexpr int FG_GROUP_M = 8;           // row tiles that are walked together down the columns: their A tiles stay in L2 while B passes once
constexpr int FG_SMEM = 192 * 1024;     // ring of stages

template <int CG, int BN>
struct FgShape {
    static constexpr uint32_t A_BYTES = FG_BM * FG_BK * 2, B_ROWS = BN / CG, B_BYTES = B_ROWS * FG_BK * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int NS = FG_SMEM / STAGE;
};

struct FgParams {
    FgArgs g;
    int m_tiles, n_tiles, k_blocks;
    int vec_out, vec_res, vec_z, vec_bias;  // rows allow 16-byte accesses
};

template <int CG>
__device__ __forceinline__ void tc_mma_f16(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(adesc), "l"(bdesc),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(adesc), "l"(bdesc),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
}
// the MMAs issued so far, when done, arrive on this barrier (CG = 2: on the barrier at the same place in both CTAs of the pair)
template <int CG>
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
    else
        tc_commit(bar);
}
template <int CG>
__device__ __forceinline__ void tmem_alloc_all(uint32_t smem_dst) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_dst) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(smem_dst, 512);
        tmem_relinquish();
    }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc_all(uint32_t taddr) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
    else tmem_dealloc(taddr, 512);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of the same shared-memory location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// a box into this CTA's shared memory, its bytes counted on a barrier that may lie in the other CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(tm), "r"(x), "r"(y),
                 "r"(cluster_bar)
                 : "memory");
}

// MN-major operand tile with the 128-byte swizzle: boxes of 64 rows-of-the-operand x 64 k, [box][k][64]; 8 k are 1024 bytes apart (stride
// offset), the next 64 operand rows one box further (leading offset).
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// instruction descriptor of kind::f16: fp32 accumulators, both operands of one 16-bit type, M = 128
__device__ __forceinline__ uint32_t f16_idesc(int is_f16, int a_mn, int b_mn, int m, int n) {
    const uint32_t t = is_f16 ? 0u : 1u;
    return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

struct Tile { int m, n; };
__device__ __forceinline__ Tile tile_at(int i, int m_tiles, int n_tiles) {
    const int per = FG_GROUP_M * n_tiles, g = i / per, first = g * FG_GROUP_M;
    const int gm = min(FG_GROUP_M, m_tiles - first), r = i - g * per;
    return {first + r % gm, r / gm};
}

template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vec, int n, float (&v)[16]) {
    if (vec && n >= 16) {
        load8<T>(p, *reinterpret_cast<float(*)[8]>(&v[0]));
        load8<T>(p + 8, *reinterpret_cast<float(*)[8]>(&v[8]));
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store16(T* p, bool vec, int n, const float (&v)[16]) {
    if (vec && n >= 16) {
        store8<T>(p, *reinterpret_cast<const float(*)[8]>(&v[0]));
        store8<T>(p + 8, *reinterpret_cast<const float(*)[8]>(&v[8]));
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

// 16 columns of one output row
template <typename T>
__device__ __forceinline__ void epilogue16(const FgParams& P, long long row, int col, const uint32_t (&acc)[16]) {
    const FgArgs& g = P.g;
    const int n = g.N - col;
    float z[16];
    if (g.bias) {
        load16<T>(reinterpret_cast<const T*>(g.bias) + col, P.vec_bias, n, z);
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] += __uint_as_float(acc[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = __uint_as_float(acc[i]);
    }
    if (g.z_out) store16<float>(g.z_out + row * g.z_ld + col, P.vec_z, n, z);
    if (g.act != ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = act_fwd(g.act, z[i]);
    }
    if (g.res) {
        float r[16];
        load16<T>(reinterpret_cast<const T*>(g.res) + row * g.res_ld + col, P.vec_res, n, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] += r[i];
    }
    store16<T>(reinterpret_cast<T*>(g.out) + row * g.out_ld + col, P.vec_out, n, z);
}

// 16 columns of one row of the gated product: gate and up accumulators of output columns col ..
template <typename T>
__device__ __forceinline__ void epilogue16_dual(const FgParams& P, long long row, int col, const uint32_t (&ga)[16], const uint32_t (&ua)[16]) {
    const FgArgs& g = P.g;
    const int n = g.inter - col;
    float a[16], b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) { a[i] = __uint_as_float(ga[i]); b[i] = __uint_as_float(ua[i]); }
    if (g.z_out) {
        float* z = g.z_out + row * g.z_ld + col;
        store16<float>(z, P.vec_z, n, a);
        store16<float>(z + g.inter, P.vec_z, n, b);
    }
    if (g.limit > 0.f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {  // comparisons that a NaN passes through
            a[i] = a[i] > g.limit ? g.limit : a[i];
            b[i] = b[i] > g.limit ? g.limit : (b[i] < -g.limit ? -g.limit : b[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) a[i] = act_fwd(g.act, a[i]) * b[i];
    store16<T>(reinterpret_cast<T*>(g.out) + row * g.out_ld + col, P.vec_out, n, a);
}

template <typename T, int CG, int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(FG_THREADS, 1) fg_gemm_kernel(const FgParams P, const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b) {
    using S = FgShape<CG, BN>;
    constexpr int NS = S::NS;
    extern __shared__ __align__(1024) uint8_t smem_dyn[];
    __shared__ __align__(8) unsigned long long bars[2 * NS + 4];  // full[s], empty[s], acc_full[2], acc_empty[2]
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;  // the first CTA of a pair issues the MMAs; full[] and acc_empty[] are used there
    uint8_t* ring = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    auto bar_full = [&](int s) { return smem_u32(&bars[s]); };
    auto bar_empty = [&](int s) { return smem_u32(&bars[NS + s]); };
    auto bar_acc_full = [&](int b) { return smem_u32(&bars[2 * NS + b]); };
    auto bar_acc_empty = [&](int b) { return smem_u32(&bars[2 * NS + 2 + b]); };
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < NS; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(bar_acc_full(b), 1); mbar_init(bar_acc_empty(b), 8 * CG); }
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc_all<CG>(smem_u32(&tmem_base_sh));
    tc_fence_before();
    __syncwarp();
    if constexpr (CG == 2) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;
    pdl_wait();
    pdl_launch_dependents();
    const FgArgs& g = P.g;
    const int tiles = P.m_tiles * P.n_tiles, first = blockIdx.x / CG, step = gridDim.x / CG;

    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tm_a);
            tma_prefetch_desc(&tm_b);
            uint32_t n = 0;
            for (int i = first; i < tiles && !abort_flag; i += step) {
                const Tile t = tile_at(i, P.m_tiles, P.n_tiles);
                const int m0 = (t.m * CG + (int)rank) * FG_BM;
                // the two halves of the B tile: consecutive rows, or gate rows and up rows; a CTA of a pair loads one of them
                const int h0 = g.dual ? t.n * (BN / 2) : t.n * BN, h1 = g.dual ? g.inter + h0 : h0 + BN / 2;
                const int n0 = rank ? h1 : h0;
                for (int kb = 0; kb < P.k_blocks; ++kb, ++n) {
                    const uint32_t s = n % NS, ph = (n / NS) & 1;
                    if (!mbar_wait(bar_empty(s), ph ^ 1, &abort_flag, &g_fg_error, 1)) break;
                    const uint32_t da = smem_u32(ring + (size_t)s * S::STAGE), db = da + S::A_BYTES;
                    const int k0 = kb * FG_BK;
                    if (rank == 0) mbar_expect_tx(bar_full(s), CG * S::STAGE);
                    const uint32_t bar = CG == 2 ? map_rank(bar_full(s), 0) : bar_full(s);
                    auto load = [&](uint32_t dst, const CUtensorMap* tm, int x, int y) {
                        if constexpr (CG == 2) tma_load_2d_pair(dst, tm, x, y, bar);
                        else tma_load_2d(dst, tm, x, y, bar);
                    };
                    if constexpr (A_MN) {
#pragma unroll
                        for (int q = 0; q < FG_BM / 64; ++q) load(da + q * 8192, &tm_a, m0 + q * 64, k0);
                    } else {
                        load(da, &tm_a, k0, m0);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int q = 0; q < (int)S::B_ROWS / 64; ++q) load(db + q * 8192, &tm_b, n0 + q * 64, k0);
                    } else {
                        load(db, &tm_b, k0, n0);
                        if constexpr (CG == 1) load(db + S::B_BYTES / 2, &tm_b, k0, h1);
                    }
                }
            }
            // every load issued above must have landed before the CTA may exit (the second CTA of a pair is kept by the cluster barrier below)
            for (int k = 0; rank == 0 && k < NS && k < (int)n; ++k) {
                const uint32_t m = n - 1 - k, s = m % NS, ph = (m / NS) & 1;
                const unsigned long long t0 = global_timer_ns();
                while (!mbar_test(bar_full(s), ph))
                    if (global_timer_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(&g_fg_error, 0, 2); break; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = f16_idesc(g.is_f16, A_MN, B_MN, FG_BM * CG, BN);
            uint32_t n = 0, it = 0;
            for (int i = first; i < tiles && !abort_flag; i += step, ++it) {
                const uint32_t buf = it & 1, aph = (it >> 1) & 1;
                if (!mbar_wait(bar_acc_empty(buf), aph ^ 1, &abort_flag, &g_fg_error, 11)) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * BN;
                for (int kb = 0; kb < P.k_blocks; ++kb, ++n) {
                    const uint32_t s = n % NS, ph = (n / NS) & 1;
                    if (!mbar_wait(bar_full(s), ph, &abort_flag, &g_fg_error, 12)) break;
                    tc_fence_after();
                    const uint32_t sa = smem_u32(ring + (size_t)s * S::STAGE), sb = sa + S::A_BYTES;
                    const uint64_t da = A_MN ? desc_mn_sw128(sa) : desc_sw128(sa), db = B_MN ? desc_mn_sw128(sb) : desc_sw128(sb);
#pragma unroll
                    for (int j = 0; j < FG_BK / 16; ++j)  // 16 k further: 32 bytes inside the swizzled row, or two groups of 8 k (2048 bytes)
                        tc_mma_f16<CG>(d, da + j * (A_MN ? 128 : 2), db + j * (B_MN ? 128 : 2), idesc, (kb | j) != 0);
                    tc_commit_pair<CG>(bar_empty(s));
                }
                tc_commit_pair<CG>(bar_acc_full(buf));
            }
        }
    } else if (warp >= 4) {
        const int q = warp & 3, half = warp >= 8 ? 1 : 0;
        uint32_t it = 0;
        for (int i = first; i < tiles; i += step, ++it) {
            const Tile t = tile_at(i, P.m_tiles, P.n_tiles);
            const uint32_t buf = it & 1, aph = (it >> 1) & 1;
            if (!mbar_wait(bar_acc_full(buf), aph, &abort_flag, &g_fg_error, 21)) break;
            tc_fence_after();
            const long long row = (long long)(t.m * CG + (int)rank) * FG_BM + q * 32 + lane;
            const uint32_t t0 = tmem + ((uint32_t)(q * 32) << 16) + buf * BN;
            if (g.dual) {
                for (int c = half * (BN / 4); c < (half + 1) * (BN / 4); c += 16) {
                    uint32_t a[16], b[16];
                    tc_ld16(t0 + c, a);
                    tc_ld16(t0 + BN / 2 + c, b);
                    tc_wait_ld();
                    const int col = t.n * (BN / 2) + c;
                    if (row < g.M && col < g.inter) epilogue16_dual<T>(P, row, col, a, b);
                }
            } else {
                for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 16) {
                    uint32_t a[16];
                    tc_ld16(t0 + c, a);
                    tc_wait_ld();
                    const int col = t.n * BN + c;
                    if (row < g.M && col < g.N) epilogue16<T>(P, row, col, a);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) mbar_arrive_cluster(map_rank(bar_acc_empty(buf), 0));
                else mbar_arrive(bar_acc_empty(buf));
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    if constexpr (CG == 2) {
        cluster_sync();  // neither CTA leaves while the other may still signal its barriers or read its shared memory
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_all<CG>(tmem);
    }
}

// ------------------------------------------------------------------ host
int sm_count();

static int fg_tmap(CUtensorMap* tm, const FgOperand& o, int is_f16, long long rows, long long k, uint32_t box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return (int)cudaErrorNotSupported;
    cuuint64_t dims[2] = {(cuuint64_t)(o.mn_major ? rows : k), (cuuint64_t)(o.mn_major ? k : rows)};
    cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
    cuuint32_t box[2] = {64, o.mn_major ? 64u : box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(tm, is_f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(o.base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <typename T, int CG, int BN, bool A_MN, bool B_MN>
static int fg_run(FgParams& P, cudaStream_t stream) {
    using S = FgShape<CG, BN>;
    const FgArgs& g = P.g;
    P.m_tiles = (g.M + CG * FG_BM - 1) / (CG * FG_BM);
    P.n_tiles = g.dual ? (g.inter + BN / 2 - 1) / (BN / 2) : (g.N + BN - 1) / BN;
    P.k_blocks = (g.K + FG_BK - 1) / FG_BK;
    if ((long long)P.m_tiles * P.n_tiles > 0x3FFFFFFFll) return ERR_TOO_LARGE;
    alignas(64) CUtensorMap ta, tb;
    int rc = fg_tmap(&ta, g.a, g.is_f16, g.M, g.K, FG_BM);
    if (!rc) rc = fg_tmap(&tb, g.b, g.is_f16, g.N, g.K, BN / 2);
    if (rc) return rc;
    const size_t smem = (size_t)S::NS * S::STAGE + 1024;
    auto kernel = fg_gemm_kernel<T, CG, BN, A_MN, B_MN>;
    static bool attr_done[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    const int tiles = P.m_tiles * P.n_tiles, groups = sm_count() / CG;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((tiles < groups ? tiles : groups) * CG);
    cfg.blockDim = dim3(FG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CG == 2 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, P, ta, tb);
}

template <typename T, int CG, int BN>
static int fg_layouts(FgParams& P, cudaStream_t stream) {
    if (P.g.a.mn_major) return P.g.b.mn_major ? fg_run<T, CG, BN, true, true>(P, stream) : ERR_UNSUPPORTED;
    return P.g.b.mn_major ? fg_run<T, CG, BN, false, true>(P, stream) : fg_run<T, CG, BN, false, false>(P, stream);
}

template <typename T>
static int fg_dispatch(FgParams& P, cudaStream_t stream) {
    if (P.g.M <= FG_BM) return fg_layouts<T, 1, 128>(P, stream);
    return fg_layouts<T, 2, 256>(P, stream);
}

int fg_launch(const FgArgs& a, cudaStream_t stream) {
    if (!a.a.base || !a.b.base || !a.out) return ERR_BAD_ARG;
    if (a.M <= 0 || a.N <= 0 || a.K <= 0) return ERR_BAD_SHAPE;
    if (a.dual && (a.N != 2 * a.inter || a.b.mn_major)) return ERR_BAD_SHAPE;
    if (((uintptr_t)a.a.base & 15) || ((uintptr_t)a.b.base & 15) || a.a.ld % 8 || a.b.ld % 8) return ERR_BAD_ALIGN;
    if (a.a.ld < (a.a.mn_major ? a.M : a.K) || a.b.ld < (a.b.mn_major ? a.N : a.K)) return ERR_BAD_SHAPE;
    if (a.M <= FS_MAX_M && !a.a.mn_major && !a.b.mn_major) return fs_launch(a, stream);
    FgParams P{};
    P.g = a;
    auto vec = [](const void* p, long long ld) { return p && !((uintptr_t)p & 15) && ld % 8 == 0; };
    P.vec_out = vec(a.out, a.out_ld);
    P.vec_res = vec(a.res, a.res_ld);
    P.vec_z = vec(a.z_out, a.z_ld) && (!a.dual || a.inter % 8 == 0);
    P.vec_bias = vec(a.bias, 0);
    return a.is_f16 ? fg_dispatch<__half>(P, stream) : fg_dispatch<__nv_bfloat16>(P, stream);
}

int fg_device_error(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_fg_error, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    if (v) {
        int z = 0;
        cudaMemcpyToSymbol(g_fg_error, &z, sizeof(int));
    }
    *out = v;
    return 0;
}

}  // namespace b200
