// kd_gemm8.cu -- the product of two 8-bit operands (kd_fp8.cuh) on the tensor cores of sm_100a (B200):
//
//   y[m][n] = round( sum_k x[m][k] w[n][k] + bias[n] ),   x and w e4m3 codes times 2^e per 128 columns
//
// The scales are powers of two in 8 bits, which the MMA takes beside its operands (kind::mxf8f6f4.block_scale):
// it multiplies the scaled values exactly and accumulates in fp32 in TMEM, so a block of 128 columns costs no
// work outside the tensor core.  The instruction covers 32 columns and selects its scale byte by the descriptor's
// scale id; the four instructions of a block name the same byte, and one 32-bit TMEM column holds the bytes of four
// blocks (512 columns).
#include <algorithm>

#include "kd_fp8.cuh"
#include "kd_host.h"
#include "kd_internal.h"

namespace kd {
namespace {

// ------------------------------------------------------------------ primitives
// The four MMAs of a block of 128 columns, D[tmem] (+)= A * B with block scales at sa / sb in TMEM, their operands 32
// bytes of each row apart; executed by a converged warp, issued by one lane.  One warp issues all MMAs of a tile, so
// its instructions count: with an election and descriptors for each MMA, and the ring's and the parts' bookkeeping at
// run time, the loop of the pair kernel took 1,700 cycles a block where its MMAs take 768.
#define KD_MMA8_BLOCK(group)                                                                                              \
    "{\n\t.reg .pred e, p, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"                                                   \
    "elect.sync _|e, 0xffffffff;\n\t"                                                                                     \
    "setp.ne.b32 p, %6, 0;\n\t"                                                                                           \
    "setp.eq.b32 t, 0, 0;\n\t"                                                                                            \
    "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"                                                  \
    "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"                                                  \
    "@e tcgen05.mma.cta_group::" group ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t"   \
    "@e tcgen05.mma.cta_group::" group ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a1, b1, %3, [%4], [%5], t;\n\t"   \
    "@e tcgen05.mma.cta_group::" group ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a2, b2, %3, [%4], [%5], t;\n\t"   \
    "@e tcgen05.mma.cta_group::" group ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a3, b3, %3, [%4], [%5], t;\n\t}\n"
template <int kGroup>
__device__ __forceinline__ void mma8_block(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa,
                                           uint32_t sb, uint32_t accumulate) {
    if constexpr (kGroup == 1)
        asm volatile(KD_MMA8_BLOCK("1")::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
                     : "memory");
    else
        asm volatile(KD_MMA8_BLOCK("2")::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
                     : "memory");
}
#undef KD_MMA8_BLOCK
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

// 32 consecutive columns of 16 TMEM lanes spread over a warp: u[4 k .. 4 k + 1] are columns 8 k + 2 (lane % 4) and the
// next of lane taddr + lane / 4, u[4 k + 2 .. 4 k + 3] the same columns eight lanes on.
__device__ __forceinline__ void tmem_ld_spread_sync(uint32_t taddr, uint32_t* u) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr)
        : "memory");
}

template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Allows a kernel its dynamic shared memory, once on each device.
template <typename K>
cudaError_t allow_smem(K kern, int bytes, int device, PerDevice& done) {
    cudaError_t e = cudaSuccess;
    done.get(device, [&] { return (e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) == cudaSuccess; });
    return e;
}

// The output row of token m; L tokens to a sequence (all of them when the rows are evenly spaced).
__device__ __forceinline__ char* token_row(const Gemm8Params& p, int m) {
    char* y = static_cast<char*>(p.y);
    if (p.L >= p.M) return y + (long long)m * p.y_nb1;
    return y + (long long)(m / p.L) * p.y_nb2 + (long long)(m % p.L) * p.y_nb1;
}

// ------------------------------------------------------------------ few tokens
// One CTA: 128 output features (the MMA's M) x nt tokens (its N) over a range of K blocks.  With few tokens the
// weight's bytes are the work, so weights are the operand of full height and the tokens only widen the instruction.
// The K range is split over a cluster when that spreads the bytes better over the SMs; the parts are joined
// through distributed shared memory in the order of the ranks, so results do not depend on timing.
// A stage is one block of 128 columns: 16 KB of weights, nt * 128 bytes of tokens, and both scale tiles.  Shared memory
// and TMEM are taken as needed, so that CTAs with few blocks share an SM and one's copies run under another's join.
constexpr int kSWeightBytes = kGemm8BoxRows * 128;
constexpr int kSScaleBytes = 3 * 512;  // weights' tile, up to two tiles of tokens
constexpr int kSMaxStages = 12;
constexpr int kSFixed = (2 * kSMaxStages + 1) * 8 + 16 + 1024;  // barriers, TMEM address and abort flag, alignment
constexpr int kSJoinWarps = 8, kSThreads = 32 * (2 + kSJoinWarps);  // warp 0 copies, warp 1 issues MMAs, the others join
constexpr uint32_t kSScaleCols = 32;  // two sets of scale columns: 4 of the weights, 8 of the tokens

__host__ __device__ constexpr int few_stage_bytes(int nt) { return kSWeightBytes + nt * 128; }
// Stages of a CTA with nk blocks: all of them if they fit (with their scales) and room for the sums at least.
__host__ __device__ constexpr int few_stages(int nt, int nk) {
    const int fit = (232448 - kSFixed) / (few_stage_bytes(nt) + kSScaleBytes);
    const int most = fit < kSMaxStages ? fit : kSMaxStages;
    const int sums = (nt * 512 + few_stage_bytes(nt) - 1) / few_stage_bytes(nt);
    const int want = nk > sums ? nk : sums;
    return want < most ? want : most;
}
static_assert(few_stages(kGemm8MaxTokens, 1) * few_stage_bytes(kGemm8MaxTokens) >= kGemm8MaxTokens * 512, "room for the sums");
__host__ __device__ constexpr uint32_t few_tmem_cols(int nt) {
    return nt + kSScaleCols <= 64 ? 64 : (nt + kSScaleCols <= 128 ? 128 : (nt + kSScaleCols <= 256 ? 256 : 512));
}
// At least the share of the SM's 228 KB (1 KB a CTA is the system's) that the CTA takes of its 512 TMEM columns: CTAs that
// share an SM then never wait for each other's columns, which clusters that wait for their own CTAs could do for good.
constexpr int few_smem(int nt, int nk) {
    const int need = few_stages(nt, nk) * (few_stage_bytes(nt) + kSScaleBytes) + kSFixed;
    const int share = (int)few_tmem_cols(nt) * (233472 / 512) - 1024;
    return need > share ? need : share;
}

template <typename TO>
__global__ void __launch_bounds__(kSThreads)
    gemm8_few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                     const __grid_constant__ Gemm8Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const uint32_t rank = cluster_rank();
    const int n0 = (int)(blockIdx.x / p.splits) * kGemm8BoxRows;
    const int blocks = (p.K + 127) >> 7;
    const int k0 = (int)((long long)blocks * rank / p.splits), k1 = (int)((long long)blocks * (rank + 1) / p.splits);
    const int nk = k1 - k0;  // at least 1: splits <= blocks
    const int token_tiles = (p.M + 127) >> 7;
    const bool direct = p.splits == 1 && p.nt == 16;  // sums of few tokens are stored from where they are
    // the ring's size goes by the largest part, as the host's
    const int stages = few_stages(p.nt, (blocks + p.splits - 1) / p.splits);
    const uint32_t stage_bytes = few_stage_bytes(p.nt), scale_at = stages * stage_bytes;
    const uint32_t cols = few_tmem_cols(p.nt), scale_col = cols - kSScaleCols;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + scale_at + stages * kSScaleBytes);
    uint64_t* empty = full + kSMaxStages;
    uint64_t* done = empty + kSMaxStages;
    uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);
    unsigned* abort_flag = slot + 1;  // of this CTA alone
    const DevCtl ctl{p.err, abort_flag, p.wait_ns};

    auto copy_block = [&](int i, int s) {  // block i of this CTA into stage s
        const uint32_t bar = smem_u32(&full[s]), st = base + s * stage_bytes, sc = base + scale_at + s * kSScaleBytes;
        const int kb = k0 + i;
        const bool scales = i == 0 || (kb & 3) == 0;  // a scale tile covers four blocks
        mbar_arrive_expect_tx(&full[s], stage_bytes + (scales ? 512u * (1 + token_tiles) : 0u));
        tma_load_2d(st, &tmW, bar, kb * 128, n0);
        tma_load_2d(st + kSWeightBytes, &tmX, bar, kb * 128, 0);
        if (scales) {
            bulk_load(sc, p.w_scales + fp8_scale_offset(n0, kb & ~3, p.ktiles), 512, bar);
            for (int t = 0; t < token_tiles; ++t)
                bulk_load(sc + 512 * (1 + t), p.x_scales + fp8_scale_offset(128 * t, kb & ~3, p.ktiles), 512, bar);
        }
    };

    // The first stages are on their way before the CTA meets: their copies need nothing but the barriers.
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        fence_mbar_init();
        wait_for_previous();
        for (int i = 0; i < min(nk, stages); ++i) copy_block(i, i);
    }
    if (warp == 1) {
        tmem_alloc(slot, cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    launch_next();
    wait_for_previous();

    if (warp == 0) {
        for (int i = stages; i < nk; ++i) {
            const int s = i % stages;
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ((i / stages) & 1u) ^ 1u, ctl, kErrTimeoutKVEmpty))) break;
            if (lane == 0) copy_block(i, s);
            __syncwarp();
        }
    } else if (warp == 1) {
        constexpr uint32_t dhi = sw128_desc_hi(1024);
        const uint32_t idesc0 = idesc_e4m3_block(128, p.nt, 0);
        uint32_t sa = tmem + scale_col;  // the two sets differ in bit 4
        bool ok = true;
        int i = 0, s = 0, turn = 0;
        for (; i < nk; ++i) {
            const int kb = k0 + i;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full[s], turn & 1u, ctl, kErrTimeoutKVFull)))) break;
            tc_fence_after();
            if (i == 0 || (kb & 3) == 0) {
                sa ^= 16u;
                const uint32_t sc = base + scale_at + s * kSScaleBytes;
                scales_to_tmem(sa, desc_scale_tile(sc));
                for (int t = 0; t < token_tiles; ++t) scales_to_tmem(sa + 4 + 4 * t, desc_scale_tile(sc + 512 * (1 + t)));
            }
            const uint32_t idesc = idesc0 | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
            const uint32_t alo = sw128_desc_lo(base + s * stage_bytes, 16);
            const uint32_t blo = sw128_desc_lo(base + s * stage_bytes + kSWeightBytes, 16);
            mma8_block<1>(tmem, desc_join(alo, dhi), desc_join(blo, dhi), idesc, sa, sa + 4, i ? 1u : 0u);
            tc_commit(&empty[s]);
            if (++s == stages) s = 0, ++turn;
        }
        if (ok) {
            tc_commit(done);
        } else if (i > 0) {  // gave up: wait for the MMAs in flight, which read this CTA's memory
            tc_commit(done);
            mbar_wait(done, 0, ctl, kErrTimeoutDrain, false);
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;  // TMEM lanes 32 q .. of this warp, every other 16 columns
        const int f = q * 32 + lane, n = n0 + f;
        const float bias = direct && p.bias && n < p.N ? p.bias[n] : 0.0f;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0, ctl, kErrTimeoutO));
        tc_fence_after();
        if (ok && *reinterpret_cast<volatile unsigned*>(abort_flag) == 0) {
            const uint32_t src = tmem + ((uint32_t)(q * 32) << 16);
            // all copies have been consumed by completed MMAs: the stages may hold the sums [token][feature] now
            float* part = reinterpret_cast<float*>(smem);
            for (int c = half * 16; c < p.nt; c += 32) {
                float v[16];
                tmem_ld16_sync(src + c, v);
                if (direct) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (c + j < p.M && n < p.N)
                            reinterpret_cast<TO*>(token_row(p, c + j))[n] = round_to<TO>(v[j] + bias);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(c + j) * 128 + f] = v[j];
                }
            }
        }
        tc_fence_before();
    }
    if (!direct) {
        __syncwarp();
        cluster_sync_all();  // every rank's sums are in its shared memory
        if (warp >= 2) {
            // A warp adds the ranks' sums of 128 features, two tokens at a time: their reads, from the other SMs, are
            // under way together.
            const int n = n0 + lane * 4, step = p.splits * kSJoinWarps;
            float b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = p.bias && n + j < p.N ? p.bias[n + j] : 0.0f;
            for (int c0 = (int)rank + p.splits * (warp - 2); c0 < p.M; c0 += 2 * step) {
                float4 a[2];
#pragma unroll
                for (int r0 = 0; r0 < 8; r0 += 4) {
                    if (r0 >= p.splits) break;
                    float4 v[2][4];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (r0 + r < p.splits && c0 + t * step < p.M)
                                v[t][r] = ld_cluster_v4(base + (uint32_t)((c0 + t * step) * 128 + lane * 4) * 4u, (uint32_t)(r0 + r));
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (r0 == 0) a[t] = v[t][0];
#pragma unroll
                        for (int r = r0 == 0 ? 1 : 0; r < 4; ++r)
                            if (r0 + r < p.splits) a[t].x += v[t][r].x, a[t].y += v[t][r].y, a[t].z += v[t][r].z, a[t].w += v[t][r].w;
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int c = c0 + t * step;
                    if (c >= p.M) break;
                    TO* y = reinterpret_cast<TO*>(token_row(p, c)) + n;
                    const float w[4] = {a[t].x + b[0], a[t].y + b[1], a[t].z + b[2], a[t].w + b[3]};
                    if (p.y_vec && n + 4 <= p.N) {  // (32-byte aligned rows: four values are 8 or 16 aligned bytes)
                        if constexpr (sizeof(TO) == 4) *reinterpret_cast<float4*>(y) = make_float4(w[0], w[1], w[2], w[3]);
                        else *reinterpret_cast<uint2*>(y) = make_uint2(Pack2<TO>::pack(w[0], w[1]), Pack2<TO>::pack(w[2], w[3]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (n + j < p.N) y[j] = round_to<TO>(w[j]);
                    }
                }
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
        tmem_dealloc(tmem, cols);
    }
}

// ------------------------------------------------------------------ many tokens
// Tiles of 256 tokens on CTA pairs: tcgen05.mma.cta_group::2 reads 128 token rows and half of the feature rows from
// each CTA, so an operand byte is staged once for both.  A tile has one or two parts of pn features (two of 192, or
// one of 192 or 128), each an accumulator of its own in TMEM.
//
// What decides the shape, in cycles per block of 128 columns (B200, 31,744 x 4,096 x 4,096):
//   - the SM takes in at most about 58 bytes a cycle from L2 (copies alone, at any copy size): 256 x 256 tiles
//     stage 32 KB a block, 563 cycles against 512 of MMAs; 256 x 384 stage 40 KB, 706 against 768.
//   - MMAs with N = 192 run at the full rate, with N = 128 at 0.7 of it (the tokens' rows are read again too often).
//   - an accumulator is read out in some 1,500 cycles, and with one of 256 columns beside the scales there is no room
//     for another: the tensor cores paused 3,800 cycles a tile.  Two parts are read out one after the other instead:
//     at a tile's end the first part's last MMAs go first, and are read out under the second's.
constexpr int kPairM = 256, kHalfM = 128;
constexpr int kPTokenBytes = kHalfM * 128;                  // a stage is one block of 128 columns
constexpr int kPRingBytes = 5 * (kPTokenBytes + 192 * 128);  // five stages of the widest tile (more of a narrower one)
constexpr int kPMaxStages = 7;
constexpr int kPScaleBytes = 4 * 512;                       // a stage's scale tiles: of the tokens, of 384 features
constexpr int kPScaleAt = kPRingBytes;
constexpr int kPBiasAt = kPScaleAt + kPMaxStages * kPScaleBytes;
constexpr int kPBarAt = kPBiasAt + 2 * 192 * 4;
constexpr int kPNumBars = 2 * kPMaxStages + 5;              // full, empty, two accumulators' full and read, drain
constexpr int kPSlotAt = kPBarAt + kPNumBars * 8;
constexpr int kPSmem = kPSlotAt + 16 + 1024;
static_assert(kPSmem <= 232448, "shared memory budget");
// Two groups of eight epilogue warps, one for each accumulator, then the copy warp and the MMA warp.
constexpr int kPGroupWarps = 8, kPEpiWarps = 16, kPThreads = 32 * (kPEpiWarps + 2);
constexpr uint32_t kPTmemCols = 512, kPAccCols = 192;
constexpr uint32_t kPScaleCol = 384;  // two sets: 4 columns of the tokens, 12 of the features
constexpr int kBandM = 8;  // token tiles swept together, so that the tiles in flight share operands in L2

__device__ __forceinline__ uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Loads into this CTA's shared memory, counted on an mbarrier of the pair's rank 0.
__device__ __forceinline__ void tma_pair_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_pair_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// The scale tile at the same offset in both CTAs' shared memory into the same columns of both CTAs' TMEM.
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t tmem, uint64_t desc) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}\n" ::"r"(tmem),
        "l"(desc)
        : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}\n" ::"r"(
            smem_u32(bar)),
        "h"((unsigned short)0x3)
        : "memory");
}

// 32 bytes in one store: a whole sector, where two 16-byte stores reach L2 as two partial writes.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t* u) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]),
                 "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
}
// 32 consecutive columns of one row that starts on a 32-byte boundary, rounded already (two to a word in 16 bits): n0 is
// the row's first column here, N the row's length.
template <typename TO>
__device__ __forceinline__ void store_row32(TO* row, int n0, int N, const uint32_t* u) {
    constexpr int kW = 32 / sizeof(TO);  // elements of a 32-byte store
#pragma unroll
    for (int i = 0; i < 32 / kW; ++i) {
        if (n0 + (i + 1) * kW <= N) {
            st_global_v8(row + n0 + i * kW, u + 8 * i);
        } else {
#pragma unroll
            for (int j = 0; j < kW; ++j) {
                if (n0 + i * kW + j >= N) break;
                if constexpr (sizeof(TO) == 4)
                    reinterpret_cast<uint32_t*>(row)[n0 + i * kW + j] = u[8 * i + j];
                else
                    reinterpret_cast<uint16_t*>(row)[n0 + i * kW + j] = (uint16_t)(u[8 * i + (j >> 1)] >> (16 * (j & 1)));
            }
        }
    }
}
template <typename TO, int kParts, bool kWide>
__global__ void __launch_bounds__(kPThreads, 1)
    gemm8_many_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                      const __grid_constant__ CUtensorMap tmXs, const __grid_constant__ CUtensorMap tmWs,
                      const __grid_constant__ Gemm8Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPBarAt);  // rank 0's count both CTAs' bytes
    uint64_t* empty = full + kPMaxStages;                          // each CTA's: its stage may be refilled
    uint64_t* acc_full = empty + kPMaxStages;                      // [2]
    uint64_t* acc_read = acc_full + 2;                             // [2], rank 0's: both CTAs have read the accumulator
    uint64_t* drain = acc_read + 2;
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + kPSlotAt);
    unsigned* abort_flag = slot + 1;
    const DevCtl ctl{p.err, abort_flag, p.wait_ns};
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int pn = p.nt, bn = pn * kParts;
    const int m_tiles = (p.M + kPairM - 1) / kPairM, n_tiles = (p.N + bn - 1) / bn;
    const long long tiles = (long long)m_tiles * n_tiles;
    const int blocks = (p.K + 127) >> 7;
    const uint32_t part_bytes = (uint32_t)pn * 64u;  // pn / 2 feature rows of 128 bytes
    const uint32_t stage_bytes = kPTokenBytes + (uint32_t)kParts * part_bytes;
    const uint32_t stages = min((uint32_t)kPRingBytes / stage_bytes, (uint32_t)kPMaxStages);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPMaxStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_read[i], 2 * kPGroupWarps);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kPEpiWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(kPTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t full0 = map_to_rank(smem_u32(full), 0);
    const uint32_t acc_read0 = map_to_rank(smem_u32(acc_read), 0);
    launch_next();
    wait_for_previous();

    auto tile_at = [&](long long t, int& mt, int& nt) {
        const long long band = t / ((long long)kBandM * n_tiles);
        const int first = (int)band * kBandM, gm = min(kBandM, m_tiles - first);
        const int within = (int)(t - band * kBandM * n_tiles);
        mt = first + within % gm;
        nt = within / gm;
    };

    if (warp == kPEpiWarps) {
        // ------------------------------------------------------------ copies (both CTAs)
        constexpr uint32_t scale_bytes = 512u * (kParts + 2);
        uint32_t s = 0, turn = 0, total = 0;
        bool ok = true;
        for (long long t = pair; t < tiles && ok; t += npairs) {
            int mt, nt;
            tile_at(t, mt, nt);
            const int m0 = mt * kPairM + (int)rank * kHalfM, n0 = nt * bn;
            for (int kb = 0; kb < blocks; ++kb, ++total) {
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (turn & 1u) ^ 1u, ctl, kErrTimeoutKVEmpty)))) break;
                if (lane == 0) {
                    const bool scales = (kb & 3) == 0;  // a scale tile covers four blocks
                    const uint32_t a = base + s * stage_bytes, bar = full0 + 8u * s;
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * (stage_bytes + (scales ? scale_bytes : 0u)));
                    tma_pair_2d(a, &tmX, bar, kb * 128, m0);
#pragma unroll
                    for (int h = 0; h < kParts; ++h)
                        tma_pair_2d(a + kPTokenBytes + h * part_bytes, &tmW, bar, kb * 128, n0 + h * pn + (int)rank * (pn / 2));
                    if (scales) {
                        const uint32_t sc = base + kPScaleAt + s * kPScaleBytes;
                        tma_pair_3d(sc, &tmXs, bar, 0, kb >> 2, m0 >> 7);
                        tma_pair_3d(sc + 512, &tmWs, bar, 0, kb >> 2, n0 >> 7);
                    }
                }
                __syncwarp();
                if (++s == stages) s = 0, ++turn;
            }
        }
        // wait for the releases of the last stages: nothing may be addressed to this CTA when it leaves
        for (uint32_t k = 0; ok && k < min(total, stages); ++k) {
            if (s == 0) s = stages, --turn;
            --s;
            ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], turn & 1u, ctl, kErrTimeoutDrain));
        }
    } else if (warp == kPEpiWarps + 1) {
        // ------------------------------------------------------------ MMAs (rank 0)
        if (rank == 0) {
            constexpr uint32_t dhi = sw128_desc_hi(1024);
            constexpr uint32_t kNextId = (1u << 4) | (1u << 29);  // the next scale byte of both operands
            const uint32_t idesc0 = idesc_e4m3_block(kPairM, pn, 0);
            const uint32_t lo0 = sw128_desc_lo(base, 16), lo_step = stage_bytes >> 4, part_lo = part_bytes >> 4;
            // a part's first feature within the copied tiles, in columns of 32 features (even: multiples of 64)
            const uint32_t part_col = (uint32_t)pn / 32u;
            uint32_t s = 0, turn = 0, lo = lo0;            // the ring's next stage: its index, turn and descriptor word
            uint32_t sa = tmem + kPScaleCol;               // the scale set in use; the two differ in bit 4
            uint32_t reads = 0;                            // tiles whose accumulators (two parts) / tile (one) went out
            bool ok = true, issued = false;
            // Waits for the next stage and copies its scales, when it brings some.
            auto take = [&](int i) {
                if (!__all_sync(0xffffffffu, mbar_wait(&full[s], turn & 1u, ctl, kErrTimeoutKVFull))) return false;
                tc_fence_after();
                if ((i & 3) == 0) {
                    sa ^= 16u;
                    const uint32_t sc = base + kPScaleAt + s * kPScaleBytes;
#pragma unroll
                    for (int j = 0; j < 2 + kParts; ++j) scales_to_tmem_pair(sa + 4 * j, desc_scale_tile(sc + 512 * j));
                }
                return true;
            };
            auto advance = [&] {
                lo += lo_step;
                if (++s == stages) s = 0, ++turn, lo = lo0;
            };
            auto part = [&](int i, int h, uint32_t acc, uint32_t stage_lo, uint32_t set, uint32_t col) {
                mma8_block<2>(tmem + acc * kPAccCols, desc_join(stage_lo, dhi),
                                desc_join(stage_lo + (kPTokenBytes >> 4) + h * part_lo, dhi), idesc0 + (uint32_t)(i & 3) * kNextId,
                                set, set + 4 + col + h * part_col, i ? 1u : 0u);
            };
            // Two blocks from i (or one, at the end of a short row), the first part of both before the second's.
            auto part_by_part = [&](int i, int n, bool first, bool last) {
                const uint32_t s0 = s, set0 = sa ^ ((i & 3) == 0 ? 16u : 0u), l0 = lo;
                if (!take(i)) return false;
                part(i, 0, 0, l0, set0, 0);
                issued = true;
                advance();
                const uint32_t s1 = s, l1 = lo;
                if (n == 2) {
                    if (!take(i + 1)) return false;
                    part(i + 1, 0, 0, l1, sa, 0);
                    advance();
                }
                if (last) commit_pair(&acc_full[0]);
                if (first && reads) {
                    if (!__all_sync(0xffffffffu, mbar_wait(&acc_read[1], (reads - 1) & 1u, ctl, kErrTimeoutO))) return false;
                    tc_fence_after();
                }
                part(i, 1, 1, l0, set0, 0);
                commit_pair(&empty[s0]);
                if (n == 2) {
                    part(i + 1, 1, 1, l1, sa, 0);
                    commit_pair(&empty[s1]);
                }
                if (last) commit_pair(&acc_full[1]);
                return true;
            };
            for (long long t = pair; t < tiles && ok; t += npairs, ++reads) {
                if constexpr (kParts == 2) {
                    if (reads && !(ok = __all_sync(0xffffffffu, mbar_wait(&acc_read[0], (reads - 1) & 1u, ctl, kErrTimeoutO))))
                        break;
                    tc_fence_after();
                    if (!(ok = part_by_part(0, min(blocks, 2), true, blocks <= 2))) break;
                    if (blocks == 3) ok = part_by_part(2, 1, false, true);
                    if (blocks <= 3) continue;
                    for (int i = 2; i < blocks - 2; ++i) {
                        if (!(ok = take(i))) break;
                        part(i, 0, 0, lo, sa, 0);
                        part(i, 1, 1, lo, sa, 0);
                        commit_pair(&empty[s]);
                        advance();
                    }
                    ok = ok && part_by_part(blocks - 2, 2, false, true);
                } else {
                    int mt, nt;
                    tile_at(t, mt, nt);
                    const uint32_t col = (uint32_t)((nt * bn) & 127) / 32u, acc = reads & 1u;
                    if (reads >= 2 &&
                        !(ok = __all_sync(0xffffffffu, mbar_wait(&acc_read[acc], ((reads >> 1) - 1) & 1u, ctl, kErrTimeoutO))))
                        break;
                    tc_fence_after();
                    for (int i = 0; i < blocks; ++i) {
                        if (!(ok = take(i))) break;
                        part(i, 0, acc, lo, sa, col);
                        issued = true;
                        commit_pair(&empty[s]);
                        advance();
                    }
                    if (ok) commit_pair(&acc_full[acc]);
                }
            }
            if (!ok && issued) {  // gave up: wait until every MMA issued so far has retired
                commit_pair(drain);
                mbar_wait(drain, 0, ctl, kErrTimeoutDrain, false);
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue: bias, rounding, stores
        const int g = warp / kPGroupWarps;                // the accumulator of this group
        const int half = (warp >> 2) & 1, wc = pn / 2;    // columns half * wc .. of the part
        const uint32_t src = tmem + ((uint32_t)((warp & 3) * 32) << 16) + g * kPAccCols + (uint32_t)(half * wc);
        float* bias = reinterpret_cast<float*>(smem + kPBiasAt) + g * 192;
        uint32_t uses = 0, tc = 0;
        for (long long t = pair; t < tiles; t += npairs, ++tc) {
            if (kParts == 1 && (int)(tc & 1u) != g) continue;
            int mt, nt;
            tile_at(t, mt, nt);
            const int np = nt * bn + (kParts == 2 ? g * pn : 0);  // the part's first feature
            {  // its bias, while the MMAs run
                const int i = threadIdx.x - g * (32 * kPGroupWarps);
                if (uses) named_bar_sync(1 + g, 32 * kPGroupWarps);
                if (i < pn) bias[i] = p.bias && np + i < p.N ? p.bias[np + i] : 0.0f;
                named_bar_sync(1 + g, 32 * kPGroupWarps);
            }
            // After a wait gave up the group still goes through its tiles, without waiting again: its warps meet at the
            // named barrier, so none may leave alone.
            const bool ok = __all_sync(0xffffffffu, *reinterpret_cast<volatile unsigned*>(abort_flag) == 0 &&
                                                        mbar_wait(&acc_full[g], uses & 1u, ctl, kErrTimeoutO));
            tc_fence_after();
            ++uses;
            // kWide, rows on 32-byte boundaries: a lane takes a row.  Other rows are written in pairs of columns, and
            // lanes that each wrote a row of their own would touch 32 rows with every store (30,952 x 8,194 x 1,382 bf16:
            // 2,366 us against 426): there four lanes take eight neighbouring columns of a row.
            constexpr int kWords = sizeof(TO) == 4 ? 32 : 16;
            uint32_t u[3 * kWords];
            if (ok) {
#pragma unroll
                for (int c = 0; c < 3; ++c) {
                    if (32 * c < wc) {
                        uint32_t x[32];
                        const float* b = bias + half * wc + 32 * c;
                        if constexpr (kWide) {
                            tmem_ld32_sync(src + 32 * c, x);
                        } else {
                            tmem_ld_spread_sync(src + 32 * c, x);
                            tmem_ld_spread_sync(src + (16u << 16) + 32 * c, x + 16);
                        }
                        // value j of a lane: column j, or with four lanes to a row 8 (j / 4 % 4) + 2 (lane % 4) + j % 2
                        auto sum = [&](int j) {
                            return __uint_as_float(x[j]) + b[kWide ? j : 8 * (j >> 2 & 3) + 2 * (lane & 3) + (j & 1)];
                        };
                        if constexpr (sizeof(TO) == 4) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) u[c * kWords + j] = __float_as_uint(sum(j));
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) u[c * kWords + j] = Pack2<TO>::pack(sum(2 * j), sum(2 * j + 1));
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(acc_read0 + 8u * g);
            const int m0 = mt * kPairM + (int)rank * kHalfM + (warp & 3) * 32, n = np + half * wc;
            if constexpr (kWide) {
                if (ok && m0 + lane < p.M) {
                    TO* row = reinterpret_cast<TO*>(token_row(p, m0 + lane));
#pragma unroll
                    for (int c = 0; c < 3; ++c)
                        if (32 * c < wc && n + 32 * c < p.N) store_row32(row, n + 32 * c, p.N, u + c * kWords);
                }
            } else if (ok) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // rows lane / 4 + 8 j of the warp's 32
                    const int m = m0 + (lane >> 2) + 8 * j;
                    const bool live = m < p.M;
                    TO* row = reinterpret_cast<TO*>(token_row(p, live ? m : 0));
                    // words of two 16-bit columns whose row starts between two words are shifted by one column: each lane
                    // takes its second column and the first of the next lane's (of the next eight columns' first lane)
                    const bool shift = sizeof(TO) == 2 && (reinterpret_cast<uintptr_t>(row) & 2u) != 0;
                    constexpr int kGroups = 12;  // of eight columns
                    auto word = [&](int g) { return u + (g >> 2) * kWords + (16 * (j >> 1) + 4 * (g & 3) + 2 * (j & 1)) * kWords / 32; };
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        if (8 * g >= wc) break;
                        const int col = n + 8 * g + 2 * (lane & 3);
                        if constexpr (sizeof(TO) == 2) {
                            const bool last = 8 * (g + 1) >= wc;
                            const uint32_t mine = *word(g), give = (lane & 3) == 0 && !last ? *word(g + 1 < kGroups ? g + 1 : g) : mine;
                            const uint32_t next = __shfl_sync(0xffffffffu, give, (lane & ~3) | ((lane + 1) & 3));
                            uint16_t* r16 = reinterpret_cast<uint16_t*>(row);
                            if (!live) continue;
                            if (!shift) {
                                if (col + 2 <= p.N) *reinterpret_cast<uint32_t*>(r16 + col) = mine;
                                else if (col < p.N) r16[col] = (uint16_t)mine;
                            } else {
                                if (g == 0 && (lane & 3) == 0 && col < p.N) r16[col] = (uint16_t)mine;
                                if (col + 3 <= p.N && !(last && (lane & 3) == 3))
                                    *reinterpret_cast<uint32_t*>(r16 + col + 1) = (mine >> 16) | (next << 16);
                                else if (col + 2 <= p.N) r16[col + 1] = (uint16_t)(mine >> 16);
                            }
                        } else if (live) {
                            const uint32_t* w = word(g);
                            uint32_t* r32 = reinterpret_cast<uint32_t*>(row);
                            if (p.y_pair && col + 2 <= p.N) {
                                *reinterpret_cast<uint2*>(r32 + col) = make_uint2(w[0], w[1]);
                            } else {
                                if (col < p.N) r32[col] = w[0];
                                if (col + 1 < p.N) r32[col + 1] = w[1];
                            }
                        }
                    }
                }
            }
            __syncwarp();
        }
    }
    // After a wait gave up, copies may still be landing: give them time before the memory is released.
    __syncwarp();
    if (threadIdx.x == 0 && *reinterpret_cast<volatile unsigned*>(abort_flag)) {
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 50000ull) {
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();  // no CTA leaves while its partner may still signal its barriers
    if (warp == kPEpiWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kPTmemCols) : "memory");
    }
}

template <typename TO, int kParts, bool kWide>
cudaError_t many_launch(const CUtensorMap* tm, const Gemm8Params& p, int num_sms, cudaStream_t st) {
    auto kern = gemm8_many_kernel<TO, kParts, kWide>;
    static PerDevice ready, pairs;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = allow_smem(kern, kPSmem, device, ready);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)((p.M + kPairM - 1) / kPairM) * ((p.N + p.nt * p.parts - 1) / (p.nt * p.parts));
    // pairs that can be resident at one time
    const int resident = pairs.get(device, [&] {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3((unsigned)(2 * (num_sms / 2)));
        cfg.blockDim = dim3(kPThreads);
        cfg.dynamicSmemBytes = kPSmem;
        cfg.stream = st;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
        return e == cudaSuccess ? n : 0;
    });
    if (resident <= 0) return e != cudaSuccess ? e : cudaErrorInvalidConfiguration;
    return launch_following(kern, dim3((unsigned)(2 * (tiles < resident ? tiles : resident))), kPThreads, kPSmem, 2, st, tm[0],
                            tm[1], tm[2], tm[3], p);
}

template <typename TO>
cudaError_t many_typed(const CUtensorMap* tm, const Gemm8Params& p, int num_sms, cudaStream_t st) {
    if (p.y_vec) return p.parts == 2 ? many_launch<TO, 2, true>(tm, p, num_sms, st) : many_launch<TO, 1, true>(tm, p, num_sms, st);
    return p.parts == 2 ? many_launch<TO, 2, false>(tm, p, num_sms, st) : many_launch<TO, 1, false>(tm, p, num_sms, st);
}

template <typename TO>
cudaError_t few_typed(const CUtensorMap& tmX, const CUtensorMap& tmW, const Gemm8Params& p, cudaStream_t st) {
    auto kern = gemm8_few_kernel<TO>;
    static PerDevice ready;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = allow_smem(kern, 232448, device, ready);
    if (e != cudaSuccess) return e;
    return launch_following(kern, dim3((unsigned)((p.N + kGemm8BoxRows - 1) / kGemm8BoxRows) * (unsigned)p.splits), kSThreads,
                            few_smem(p.nt, ((p.K + 127) / 128 + p.splits - 1) / p.splits), (unsigned)p.splits, st, tmX, tmW, p);
}

}  // namespace

// Up to 256 tokens (the MMA's largest N) the weight is the operand of full height: 256 x 4,096 x 4,096 takes 13.7 us so and
// 16.0 in pairs of CTAs, 200 x 16,384 x 4,096 22.8 and 24.6; one token 7.3 and 16.6.  More would need the weight twice.
// Few tokens (at most 256): all of them in one tile, in steps of 16; K split over up to 8 CTAs (the portable cluster
// size) as far as all CTAs run at one time.  (More and shorter CTAs, 3 to 7 to an SM, were slower: 16,384 x 4,096 x
// one token 14.5 us unsplit, 19.3 us in two parts, 26 us in four.)
// Many tokens: the tile whose rounds over the SM pairs add up to the least, by the cost of a block of 128 columns (MMAs
// for two parts of 192, copies for one of 192 or 128, as measured above) and 1,000 cycles a tile.  The sums rank the
// tiles, they are not times: 1,999 tokens x 1,792 columns f16 take 29, 47 and 62 thousand cycles in one, two and three
// rounds of 2 x 192 (850 a block, 6,000 a round and 11,000 a launch) where the sums are 12, 23 and 35, and 31,744 x 4,096 x
// 4,096 takes 579 for 486.
void gemm8_plan(Gemm8Params* p, int num_sms) {
    p->splits = p->parts = 1;
    p->many = p->M > kGemm8MaxTokens;
    const int blocks = (p->K + 127) / 128;
    if (!p->many) {
        p->nt = (p->M + 15) / 16 * 16;
        const long long tiles = (p->N + kGemm8BoxRows - 1) / kGemm8BoxRows;
        p->splits = (int)std::min<long long>(std::min(8, blocks), std::max<long long>(1, num_sms / tiles));
        return;
    }
    const struct { int parts, pn, block_cycles; } shapes[] = {{2, 192, 768}, {1, 192, 494}, {1, 128, 424}};
    const long long m_tiles = (p->M + kPairM - 1) / kPairM, pairs = num_sms / 2;
    long long best = -1;
    for (const auto& s : shapes) {
        const long long tiles = m_tiles * ((p->N + s.parts * s.pn - 1) / (s.parts * s.pn));
        const long long cost = (tiles + pairs - 1) / pairs * ((long long)blocks * s.block_cycles + 1000);
        if (best < 0 || cost < best) {
            best = cost;
            p->parts = s.parts;
            p->nt = s.pn;
        }
    }
}

cudaError_t launch_gemm8(OutType ot, const CUtensorMap* tm, const Gemm8Params& p, int num_sms, cudaStream_t st) {
    if (p.many)
        return ot == OutType::F32 ? many_typed<float>(tm, p, num_sms, st)
                                  : (ot == OutType::F16 ? many_typed<__half>(tm, p, num_sms, st)
                                                        : many_typed<__nv_bfloat16>(tm, p, num_sms, st));
    return ot == OutType::F32 ? few_typed<float>(tm[0], tm[1], p, st)
                              : (ot == OutType::F16 ? few_typed<__half>(tm[0], tm[1], p, st)
                                                    : few_typed<__nv_bfloat16>(tm[0], tm[1], p, st));
}

}  // namespace kd
