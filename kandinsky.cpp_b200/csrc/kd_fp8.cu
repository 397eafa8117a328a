// kd_fp8.cu -- writing and reading 8-bit rows (kd_fp8.cuh) on sm_100a (B200):
//
//   norm8_kernel      h = x + residual, v = h / sqrt(mean(h^2) + eps) * gain, v into 8-bit rows
//   quant8_kernel     f32 / f16 / bf16 rows into 8-bit rows
//   quant8_ggml_kernel  q8_0 / q4_0 weight rows into 8-bit rows
//   dequant8_kernel   8-bit rows back to f32 / f16 / bf16
//
// All of them move bytes and do little else: each value is read once and written once, held in registers between.
#include "kd_fp8.cuh"
#include "kd_internal.h"

namespace kd {
namespace {

constexpr int kVec = 8;         // consecutive columns of one lane: 16 lanes are one block of 128
constexpr unsigned kInfBits = 0x7F800000u;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void unpack8(const uint4& u, const __half*, float (&v)[kVec]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack8(const uint4& u, const __nv_bfloat16*, float (&v)[kVec]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

// Columns c .. c+7 of a row of K, zeros at and past K.  vec: the row starts on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int K, bool vec, float (&v)[kVec]) {
    if (vec && c + kVec <= K) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            unpack8(*reinterpret_cast<const uint4*>(row + c), row, v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = c + i < K ? to_f32(row[c + i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int c, int K, bool vec, const float (&v)[kVec]) {
    if (vec && c + kVec <= K) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4*>(row + c) = make_uint4(Pack2<T>::pack(v[0], v[1]), Pack2<T>::pack(v[2], v[3]),
                                                            Pack2<T>::pack(v[4], v[5]), Pack2<T>::pack(v[6], v[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (c + i < K) row[c + i] = from_f32<T>(v[i]);
    }
}

// One block of 128 columns, eight to a lane of a half-warp, into codes and the block's scale byte.  Lanes at and
// past K hold zeros.  A NaN or infinity becomes a NaN code and does not count for the scale.  Every lane of the
// half-warp takes part; `live` lanes write.
__device__ __forceinline__ void encode_block(const float (&v)[kVec], const Fp8Rows& o, long long row, int c,
                                             bool live) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) top = max(top, __float_as_uint(fabsf(v[i])));
#pragma unroll
    for (int s = 8; s; s >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
    float t[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) t[i] = v[i];
    // (a warp-wide vote, so that both half-warps run the shuffles of the rare path together)
    if (__any_sync(0xffffffffu, top >= kInfBits)) {
        top = 0;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const uint32_t a = __float_as_uint(fabsf(v[i]));
            if (a >= kInfBits) t[i] = __uint_as_float(0x7FFFFFFFu);
            else top = max(top, a);
        }
#pragma unroll
        for (int s = 8; s; s >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
    }
    const uint32_t byte = fp8_scale_byte(top);
    if (!live) return;
    const float inv = fp8_scale_inverse(byte);  // a power of two: the products are exact
    const uint2 codes = make_uint2(fp8_pack4(t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv),
                                   fp8_pack4(t[4] * inv, t[5] * inv, t[6] * inv, t[7] * inv));
    // rows are at least K rounded up to 16 bytes long: the eight codes from c are inside when c is below that
    if (c < o.Kp) *reinterpret_cast<uint2*>(o.codes + row * o.row_bytes + c) = codes;
    if ((c & 127) == 0 && c < o.K) o.scales[fp8_scale_offset(row, c >> 7, o.ktiles)] = (uint8_t)byte;
}

// TPR threads hold one row, VPT vectors of eight columns each: vector j of thread t is columns 8 * (j * TPR + t).
// One pass over the data: the row stays in registers between the sum of squares and the codes.
template <typename T, int VPT>
__global__ void __launch_bounds__(1024) norm8_kernel(const Norm8Params p, int tpr) {
    __shared__ float part[32];
    const int rows_per_cta = blockDim.x / tpr;
    const int sub = threadIdx.x / tpr, t = threadIdx.x % tpr;
    const long long row = (long long)blockIdx.x * rows_per_cta + sub;
    const bool live = row < p.out.rows;
    const long long m = live ? row : p.out.rows - 1;  // a row past the end repeats the last one and writes nothing
    const int K = p.out.K;
    const long long n = m / p.L, l = m % p.L;
    const T* x = reinterpret_cast<const T*>(static_cast<const char*>(p.x) + n * p.x_nb2 + l * p.x_nb1);
    const T* r = p.r ? reinterpret_cast<const T*>(static_cast<const char*>(p.r) + n * p.r_nb2 + l * p.r_nb1) : nullptr;
    T* h = p.h ? reinterpret_cast<T*>(static_cast<char*>(p.h) + n * p.h_nb2 + l * p.h_nb1) : nullptr;
    float v[VPT][kVec];
#pragma unroll
    for (int j = 0; j < VPT; ++j) load8(x, kVec * (j * tpr + t), K, p.x_vec, v[j]);
    if (r) {
        float a[VPT][kVec];
#pragma unroll
        for (int j = 0; j < VPT; ++j) load8(r, kVec * (j * tpr + t), K, p.r_vec, a[j]);
        // the sum is rounded to the rows' type, as it is stored, and the norm is of the stored value
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[j][i] = to_f32(from_f32<T>(v[j][i] + a[j][i]));
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum = fmaf(v[j][i], v[j][i], sum);
    if (h && live) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) store8(h, kVec * (j * tpr + t), K, p.h_vec, v[j]);
    }
#pragma unroll
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (tpr > 32) {
        const int warps = tpr / 32, first = sub * warps;
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int w = 0; w < warps; ++w) sum += part[first + w];
    }
    const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)K), p.eps)));
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = kVec * (j * tpr + t);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[j][i] *= inv;
        if (p.gain) {
            float g[kVec];
            load8(p.gain, c, K, p.gain_vec, g);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[j][i] *= g[i];
        }
        encode_block(v[j], p.out, m, c, live);
    }
}

// A half-warp per block of 128 columns.
template <typename T>
__global__ void quant8_kernel(const Quant8Params p) {
    const int lane16 = threadIdx.x & 15;
    const int blocks = (p.out.K + 127) >> 7;
    const long long total = p.out.rows * blocks;
    const long long step = ((long long)gridDim.x * blockDim.x) >> 4;
    // whole warps stay in the loop: the pair's second block may be past the end
    for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 4; (i & ~1ll) < total; i += step) {
        const bool live = i < total;
        const long long row = (live ? i : total - 1) / blocks;
        const int c = (int)((live ? i : total - 1) % blocks) * 128 + lane16 * kVec;
        const T* x = reinterpret_cast<const T*>(static_cast<const char*>(p.x) + (row / p.L) * p.x_nb2 +
                                                (row % p.L) * p.x_nb1);
        float v[kVec];
        load8(x, c, p.out.K, p.x_vec, v);
        encode_block(v, p.out, row, c, live);
    }
}

// Weight rows of 32-element ggml blocks (q8_0: f16 scale and 32 int8; q4_0: f16 scale and 16 bytes, element j in
// the low nibble, j + 16 in the high one): four lanes per block of 128, one ggml block each.  Blocks are 34 or 18
// bytes long, so a lane reads 16-bit words.
__global__ void quant8_ggml_kernel(const uint8_t* w, int q4, long long row_bytes, const Fp8Rows o) {
    const int blocks = (o.K + 127) >> 7;
    const long long total = o.rows * blocks;
    const long long step = ((long long)gridDim.x * blockDim.x) >> 2;
    for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 2; (i & ~7ll) < total; i += step) {
        const bool live = i < total;
        const long long row = (live ? i : total - 1) / blocks;
        const int c = (int)((live ? i : total - 1) % blocks) * 128 + (threadIdx.x & 3) * 32;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.0f;
        if (c < o.K) {
            const uint16_t* b =
                reinterpret_cast<const uint16_t*>(w + row * row_bytes + (long long)(c >> 5) * (q4 ? 18 : 34));
            const float d = __half2float(__ushort_as_half(b[0]));
            if (q4) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned u = b[1 + j];
                    v[2 * j] = d * (float)((int)(u & 15u) - 8);
                    v[2 * j + 16] = d * (float)((int)((u >> 4) & 15u) - 8);
                    v[2 * j + 1] = d * (float)((int)((u >> 8) & 15u) - 8);
                    v[2 * j + 17] = d * (float)((int)(u >> 12) - 8);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const unsigned u = b[1 + j];
                    v[2 * j] = d * (float)(int8_t)(u & 255u);
                    v[2 * j + 1] = d * (float)(int8_t)(u >> 8);
                }
            }
        }
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const uint32_t a = __float_as_uint(fabsf(v[j]));
            if (a >= kInfBits) v[j] = __uint_as_float(0x7FFFFFFFu);  // a block whose f16 scale is not finite
            else top = max(top, a);
        }
#pragma unroll
        for (int s = 2; s; s >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
        const uint32_t byte = fp8_scale_byte(top);
        const float inv = fp8_scale_inverse(byte);
        if (!live || c >= o.K) continue;  // (K is a multiple of 32: a ggml block is wholly inside)
        uint4* dst = reinterpret_cast<uint4*>(o.codes + row * o.row_bytes + c);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* a = v + 16 * q + 4 * j;
                u[j] = fp8_pack4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
            }
            dst[q] = make_uint4(u[0], u[1], u[2], u[3]);
        }
        if ((c & 127) == 0) o.scales[fp8_scale_offset(row, c >> 7, o.ktiles)] = (uint8_t)byte;
    }
}

// Eight codes per thread.
template <typename T>
__global__ void dequant8_kernel(const Dequant8Params p) {
    const int per_row = (p.in.K + kVec - 1) / kVec;
    const long long total = p.in.rows * per_row;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (long long)gridDim.x * blockDim.x) {
        const long long row = i / per_row;
        const int c = (int)(i % per_row) * kVec;
        const uint2 u = *reinterpret_cast<const uint2*>(p.in.codes + row * p.in.row_bytes + c);
        const float s = fp8_scale_value(p.in.scales[fp8_scale_offset(row, c >> 7, p.in.ktiles)]);
        float a[4], b[4];
        fp8_unpack4(u.x, a);
        fp8_unpack4(u.y, b);
        const float v[kVec] = {a[0] * s, a[1] * s, a[2] * s, a[3] * s, b[0] * s, b[1] * s, b[2] * s, b[3] * s};
        T* y = reinterpret_cast<T*>(static_cast<char*>(p.y) + (row / p.L) * p.y_nb2 + (row % p.L) * p.y_nb1);
        store8(y, c, p.in.K, p.y_vec, v);
    }
}

template <typename T>
cudaError_t norm8_typed(const Norm8Params& p, cudaStream_t st) {
    // up to 256 columns a warp holds a row; above, 16 (32 past 16,384) columns a thread
    const int K = p.out.K;
    int tpr = 32, vpt = K <= 256 ? 1 : (K <= 16384 ? 2 : 4);
    while (tpr * vpt * kVec < K) tpr *= 2;
    const int threads = tpr < 128 ? 128 : tpr;
    const long long ctas = (p.out.rows + threads / tpr - 1) / (threads / tpr);
    auto kern = vpt == 1 ? norm8_kernel<T, 1> : (vpt == 2 ? norm8_kernel<T, 2> : norm8_kernel<T, 4>);
    kern<<<(unsigned)ctas, threads, 0, st>>>(p, tpr);
    return cudaGetLastError();
}

unsigned grid_for(long long threads, int block, int num_sms, int per_sm) {
    long long g = (threads + block - 1) / block;
    const long long cap = (long long)num_sms * per_sm;
    return (unsigned)(g > cap ? cap : (g < 1 ? 1 : g));
}

}  // namespace

cudaError_t launch_norm8(int type, const Norm8Params& p, cudaStream_t st) {
    if (p.out.rows == 0) return cudaSuccess;
    return type == 0 ? norm8_typed<float>(p, st) : (type == 1 ? norm8_typed<__half>(p, st) : norm8_typed<__nv_bfloat16>(p, st));
}

cudaError_t launch_quant8(int type, const Quant8Params& p, int num_sms, cudaStream_t st) {
    if (p.out.rows == 0) return cudaSuccess;
    const long long threads = p.out.rows * ((p.out.K + 127) / 128) * 16;
    const unsigned g = grid_for(threads, 256, num_sms, 32);
    if (type == 0) quant8_kernel<float><<<g, 256, 0, st>>>(p);
    else if (type == 1) quant8_kernel<__half><<<g, 256, 0, st>>>(p);
    else quant8_kernel<__nv_bfloat16><<<g, 256, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_quant8_ggml(const void* w, bool q4, long long row_bytes, const Fp8Rows& out, int num_sms,
                               cudaStream_t st) {
    if (out.rows == 0) return cudaSuccess;
    const long long threads = out.rows * ((out.K + 127) / 128) * 4;
    quant8_ggml_kernel<<<grid_for(threads, 128, num_sms, 16), 128, 0, st>>>(static_cast<const uint8_t*>(w), q4 ? 1 : 0,
                                                                            row_bytes, out);
    return cudaGetLastError();
}

cudaError_t launch_dequant8(int type, const Dequant8Params& p, int num_sms, cudaStream_t st) {
    if (p.in.rows == 0) return cudaSuccess;
    const unsigned g = grid_for(p.in.rows * ((p.in.K + kVec - 1) / kVec), 256, num_sms, 32);
    if (type == 0) dequant8_kernel<float><<<g, 256, 0, st>>>(p);
    else if (type == 1) dequant8_kernel<__half><<<g, 256, 0, st>>>(p);
    else dequant8_kernel<__nv_bfloat16><<<g, 256, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace kd
