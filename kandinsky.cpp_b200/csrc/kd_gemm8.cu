// kd_gemm8.cu -- the product of two 8-bit operands (kd_fp8.cuh) on the tensor cores of sm_100a (B200):
//
//   y[m][n] = round( sum_k x[m][k] w[n][k] + bias[n] ),   x and w e4m3 codes times 2^e per 128 columns
//
// The scales are powers of two in 8 bits, which the MMA takes beside its operands (kind::mxf8f6f4.block_scale):
// it multiplies the scaled values exactly and accumulates in fp32 in TMEM, so a block of 128 columns costs no
// work outside the tensor core.  The instruction covers 32 columns and selects its scale byte by the descriptor's
// scale id; the four instructions of a block name the same byte, and one 32-bit TMEM column holds the bytes of four
// blocks (512 columns).
#include "kd_fp8.cuh"
#include "kd_internal.h"

namespace kd {
namespace {

// ------------------------------------------------------------------ primitives
// D[tmem] (+)= A * B with block scales at sa / sb in TMEM; executed by a converged warp, issued by one lane.
__device__ __forceinline__ void mma8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t sa, uint32_t sb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
// One 512-byte scale tile from shared memory into four TMEM columns (32 lanes, repeated for the four lane groups).
// tcgen05.cp and tcgen05.mma of one thread execute in the order of issue.
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint64_t desc) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}\n" ::"r"(tmem),
        "l"(desc)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
// 16 consecutive TMEM columns of this thread's lane.
__device__ __forceinline__ void tmem_ld16_sync(uint32_t taddr, float (&r)[16]) {
    uint32_t u[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __uint_as_float(u[i]);
}

template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ------------------------------------------------------------------ few tokens
// One CTA: 128 output features (the MMA's M) x nt tokens (its N) over a range of K blocks.  With few tokens the
// weight's bytes are the work, so weights are the operand of full height and the tokens only widen the instruction.
// The K range is split over a cluster when the feature tiles alone do not fill the GPU; the parts are joined
// through distributed shared memory in the order of the ranks, so results do not depend on timing.
// A stage is one block of 128 columns: 16 KB of weights, nt * 128 bytes of tokens, and both scale tiles.
constexpr int kSStages = 4;
constexpr int kSWeightBytes = kGemm8BoxRows * 128;
constexpr int kSTokenBytes = kGemm8MaxTokens * 128;
constexpr int kSScaleBytes = 3 * 512;                       // weights' tile, up to two tiles of tokens
constexpr int kSStageBytes = kSWeightBytes + kSTokenBytes;  // 48 KB
constexpr int kSScaleAt = kSStages * kSStageBytes;
constexpr int kSBarAt = kSScaleAt + kSStages * kSScaleBytes;
constexpr int kSNumBars = 2 * kSStages + 1;                 // full, empty, accumulator complete
constexpr int kSSlotAt = kSBarAt + kSNumBars * 8;           // TMEM address, abort flag
constexpr int kSSmem = kSSlotAt + 16 + 1024;
static_assert(kSSmem <= 232448, "shared memory budget");
static_assert(kGemm8MaxTokens * 128 * 4 <= kSScaleAt, "the partial sums reuse the stages");
constexpr int kSThreads = 192;  // warp 0 copies, warp 1 issues MMAs, warps 2-5 read the accumulator
constexpr uint32_t kSTmemCols = 512;
constexpr uint32_t kSScaleCol = 256;  // two sets of scale columns: 4 of the weights, 8 of the tokens

template <typename TO>
__global__ void __launch_bounds__(kSThreads, 1)
    gemm8_few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                     const __grid_constant__ Gemm8Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kSBarAt);
    uint64_t* empty = full + kSStages;
    uint64_t* done = empty + kSStages;
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + kSSlotAt);
    unsigned* abort_flag = slot + 1;  // of this CTA alone
    const DevCtl ctl{p.err, abort_flag, p.wait_ns};

    const uint32_t rank = cluster_rank();
    const int n0 = (int)(blockIdx.x / p.splits) * kGemm8BoxRows;
    const int m0 = (int)blockIdx.y * p.nt;
    const int blocks = (p.K + 127) >> 7;
    const int k0 = (int)((long long)blocks * rank / p.splits), k1 = (int)((long long)blocks * (rank + 1) / p.splits);
    const int nk = k1 - k0;  // at least 1: splits <= blocks
    const int token_tiles = (min(p.M - m0, p.nt) + 127) >> 7;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kSStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(slot, kSTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;

    if (warp == 0) {
        const uint32_t bytes = kSWeightBytes + (uint32_t)p.nt * 128u + 512u * (1 + token_tiles);
        bool ok = true;
        for (int i = 0; i < nk; ++i) {
            const int s = i % kSStages;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((i / kSStages) & 1u) ^ 1u, ctl, kErrTimeoutKVEmpty))))
                break;
            if (lane == 0) {
                const uint32_t bar = smem_u32(&full[s]), st = base + s * kSStageBytes;
                const uint32_t sc = base + kSScaleAt + s * kSScaleBytes;
                const int kb = k0 + i;
                mbar_arrive_expect_tx(&full[s], bytes);
                tma_load_2d(st, &tmW, bar, kb * 128, n0);
                tma_load_2d(st + kSWeightBytes, &tmX, bar, kb * 128, m0);
                bulk_load(sc, p.w_scales + fp8_scale_offset(n0, kb & ~3, p.ktiles), 512, bar);
                for (int t = 0; t < token_tiles; ++t)
                    bulk_load(sc + 512 * (1 + t), p.x_scales + fp8_scale_offset(m0 + 128 * t, kb & ~3, p.ktiles), 512, bar);
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        constexpr uint32_t dhi = sw128_desc_hi(1024);
        bool ok = true;
        int i = 0;
        for (; i < nk; ++i) {
            const int s = i % kSStages, kb = k0 + i;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (i / kSStages) & 1u, ctl, kErrTimeoutKVFull)))) break;
            tc_fence_after();
            const uint32_t sa = tmem + kSScaleCol + 16u * (uint32_t)((kb >> 2) & 1), sb = sa + 4;
            if (i == 0 || (kb & 3) == 0) {  // four blocks share a tile
                const uint32_t sc = base + kSScaleAt + s * kSScaleBytes;
                scales_to_tmem(sa, desc_scale_tile(sc));
                for (int t = 0; t < token_tiles; ++t) scales_to_tmem(sb + 4 * t, desc_scale_tile(sc + 512 * (1 + t)));
            }
            const uint32_t idesc = idesc_e4m3_block(128, p.nt, kb & 3);
            const uint32_t alo = sw128_desc_lo(base + s * kSStageBytes, 16);
            const uint32_t blo = sw128_desc_lo(base + s * kSStageBytes + kSWeightBytes, 16);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                mma8_ss(tmem, desc_join(alo + kk * 2, dhi), desc_join(blo + kk * 2, dhi), idesc, sa, sb,
                        (i | kk) ? 1u : 0u);
            tc_commit(&empty[s]);
        }
        if (ok) {
            tc_commit(done);
        } else if (i > 0) {  // gave up: wait for the MMAs in flight, which read this CTA's memory
            tc_commit(done);
            mbar_wait(done, 0, ctl, kErrTimeoutDrain, false);
        }
    } else {
        const int q = warp & 3;  // TMEM lanes 32 q .. of this warp
        const int f = q * 32 + lane, n = n0 + f;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0, ctl, kErrTimeoutO));
        tc_fence_after();
        if (ok && *reinterpret_cast<volatile unsigned*>(abort_flag) == 0) {
            const uint32_t src = tmem + ((uint32_t)(q * 32) << 16);
            if (p.splits == 1) {
                const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.0f;
                for (int c = 0; c < p.nt; c += 16) {
                    float v[16];
                    tmem_ld16_sync(src + c, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int m = m0 + c + j;
                        if (m < p.M && n < p.N)
                            *reinterpret_cast<TO*>(static_cast<char*>(p.y) + (m / p.L) * p.y_nb2 + (m % p.L) * p.y_nb1 +
                                                   (long long)n * sizeof(TO)) = round_to<TO>(v[j] + bias);
                    }
                }
            } else {
                // all copies have been consumed by completed MMAs: the stages hold the sums [token][feature] now
                float* part = reinterpret_cast<float*>(smem);
                for (int c = 0; c < p.nt; c += 16) {
                    float v[16];
                    tmem_ld16_sync(src + c, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(c + j) * 128 + f] = v[j];
                }
            }
        }
        tc_fence_before();
    }
    if (p.splits > 1) {
        __syncwarp();
        cluster_sync_all();  // every rank's sums are in its shared memory
        if (warp >= 2) {
            const int tokens = min(p.M - m0, p.nt);
            const int n = n0 + lane * 4;
            float b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = p.bias && n + j < p.N ? __ldg(p.bias + n + j) : 0.0f;
            for (int c = (int)rank + p.splits * (warp - 2); c < tokens; c += 4 * p.splits) {
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int r = 0; r < p.splits; ++r) {
                    const float4 v = ld_cluster_v4(base + (uint32_t)(c * 128 + lane * 4) * 4u, (uint32_t)r);
                    a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
                }
                const int m = m0 + c;
                TO* y = reinterpret_cast<TO*>(static_cast<char*>(p.y) + (m / p.L) * p.y_nb2 + (m % p.L) * p.y_nb1) + n;
                const float v[4] = {a.x + b[0], a.y + b[1], a.z + b[2], a.w + b[3]};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < p.N) y[j] = round_to<TO>(v[j]);
            }
        }
        __syncwarp();
        cluster_sync_all();  // no CTA leaves while another reads its shared memory
    }
    __syncthreads();
    // After a wait gave up, copies may still be landing: give them time before the memory is released.
    if (threadIdx.x == 0 && *reinterpret_cast<volatile unsigned*>(abort_flag)) {
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 50000ull) {
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kSTmemCols);
    }
}

template <typename TO>
cudaError_t few_typed(const CUtensorMap& tmX, const CUtensorMap& tmW, const Gemm8Params& p, cudaStream_t st) {
    auto kern = gemm8_few_kernel<TO>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)((p.N + kGemm8BoxRows - 1) / kGemm8BoxRows) * (unsigned)p.splits,
                       (unsigned)((p.M + p.nt - 1) / p.nt));
    cfg.blockDim = dim3(kSThreads);
    cfg.dynamicSmemBytes = kSSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, tmX, tmW, p);
}

}  // namespace

// Tokens per tile: all of them up to 256 (in steps of 16).  K is split while the tiles leave more than half of the
// SMs idle and each part keeps at least two blocks, over at most 8 CTAs (the portable cluster size).
void gemm8_plan(Gemm8Params* p, int num_sms) {
    p->nt = p->M >= kGemm8MaxTokens ? kGemm8MaxTokens : (p->M + 15) / 16 * 16;
    const long long tiles = (long long)((p->N + kGemm8BoxRows - 1) / kGemm8BoxRows) * ((p->M + p->nt - 1) / p->nt);
    const int blocks = (p->K + 127) / 128;
    p->splits = 1;
    while (p->splits < 8 && tiles * p->splits * 2 <= num_sms && blocks >= p->splits * 4) p->splits *= 2;
}

cudaError_t launch_gemm8(OutType ot, const CUtensorMap& tmX, const CUtensorMap& tmW, const Gemm8Params& p,
                         cudaStream_t st) {
    return ot == OutType::F32 ? few_typed<float>(tmX, tmW, p, st)
                              : (ot == OutType::F16 ? few_typed<__half>(tmX, tmW, p, st)
                                                    : few_typed<__nv_bfloat16>(tmX, tmW, p, st));
}

}  // namespace kd
