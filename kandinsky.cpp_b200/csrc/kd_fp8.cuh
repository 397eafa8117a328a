// kd_fp8.cuh -- the 8-bit row format shared by the kernels that write it (kd_fp8.cu) and the product that reads
// it (kd_gemm8.cu): e4m3 codes with one power-of-two scale per 128 columns of a row.
//
// A block's scale is 2^e with the smallest e >= -126 for which max|v| <= 448 * 2^e, held as the byte e + 127.
// A power of two costs an e4m3 code no precision (the code's own exponent absorbs it, except for values 2^-14
// and less of the block's largest, which are subnormal codes either way), multiplies without rounding, and is what
// the tensor core's block scaling takes, so the product applies it inside the MMA.
//
// The bytes lie as the tensor core wants them in TMEM: tiles of 128 rows x 4 blocks, 512 bytes each, in which row
// r's four bytes are the 32-bit word (r % 32) * 4 + r / 32.  A tile is one 16-byte-aligned bulk copy and one
// tcgen05.cp.32x128b.warpx4.
#pragma once

#include "kd_common.cuh"

namespace kd {

// Byte offset of the scale of (row, block) among the tiles; ktiles = tiles along a row (ceil(blocks / 4)).
__host__ __device__ constexpr long long fp8_scale_offset(long long row, int block, int ktiles) {
    return ((row >> 7) * ktiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// The scale byte of a block whose largest magnitude has the (finite) bit pattern `amax`.  448 = 1.75 * 2^8: the
// exponent field minus 8, plus one where the significand is above 1.75 (fraction bits above 0x600000 carry).
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax) {
    const int b = (int)((amax + 0x1FFFFFu) >> 23) - 8;
    return (uint32_t)max(b, 1);
}
// 2^(byte - 127), NaN for 255, as the tensor core takes them.  The writers make 1 .. 247; rows from elsewhere may hold 0
// (2^-127, a subnormal) and 255, where the exponent field alone would say 0 and infinity.
__device__ __forceinline__ float fp8_scale_value(uint32_t byte) {
    return __uint_as_float(byte << 23 | (byte - 1u >= 254u ? 0x400000u : 0u));
}
// Of the writers' bytes.
__device__ __forceinline__ float fp8_scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Programmatic launches: a kernel of this path may start while the one before it in the stream runs out, and sets up
// its barriers, tensor memory and registers meanwhile.  launch_next: the next one may start; called once this CTA holds
// all that it will ever ask the SM for.  wait_for_previous: everything before in the stream has finished and is visible;
// every thread calls it before it touches global memory, and then loads by plain loads: read-only ones (__ldg) ask that
// the data stay as they are for the kernel's whole time, of which the end of the kernel that writes them may be a part.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches `kern` that way, as clusters of `cluster` CTAs.
template <typename... P, typename... A>
cudaError_t launch_following(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t st,
                             const A&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Four values (already divided by the scale, |v| <= 448 or NaN) to e4m3 codes, ties to even; v0 in the low byte.
__device__ __forceinline__ uint32_t fp8_pack4(float v0, float v1, float v2, float v3) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(v0), "f"(v1), "f"(v2), "f"(v3));
    return r;
}
// Four codes to f32 (exact: e4m3 is a subset of f16).
__device__ __forceinline__ void fp8_unpack4(uint32_t c, float (&v)[4]) {
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(c));
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    v[0] = a.x;
    v[1] = a.y;
    v[2] = b.x;
    v[3] = b.y;
}

}  // namespace kd
