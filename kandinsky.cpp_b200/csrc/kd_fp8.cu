// kd_fp8.cu -- writing and reading 8-bit rows (kd_fp8.cuh) on sm_100a (B200):
//
//   norm8_kernel        h = x + residual, v = h / sqrt(mean(h^2) + eps) * gain, v into 8-bit rows
//   quant8_kernel       f32 / f16 / bf16 rows into 8-bit rows
//   quant8_ggml_kernel  q8_0 / q4_0 weight rows into 8-bit rows
//   dequant8_kernel     8-bit rows back to f32 / f16 / bf16
//
// All of them move bytes and do little else: each value is read once and written once, held in registers between.
// A warp's unit of work is 512 columns of a row: four blocks, one 32-bit word of scale bytes, sixteen columns a lane.
// Where rows start on 16-byte boundaries a lane holds sixteen consecutive columns and moves them in wide accesses;
// elsewhere (odd row lengths) lane l holds the pairs of columns 2 l, 2 l + 64, ..., so that its narrow accesses are still
// coalesced.  16-bit rows that start between two words are moved word by word all the same, shifted by one column:
// the missing half comes from the next lane.
#include <algorithm>
#include <type_traits>

#include "kd_fp8.cuh"
#include "kd_internal.h"

namespace kd {
namespace {

constexpr int kPer = 16;        // columns of a lane
constexpr int kChunk = 512;     // columns of a warp
constexpr unsigned kInfBits = 0x7F800000u;
constexpr unsigned kAll = 0xffffffffu;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Sixteen values of a lane as they lie in memory (32 or 64 bytes).
template <typename T>
struct Raw {
    static constexpr int kWords = sizeof(T) * kPer / 4;
    uint32_t w[kWords];
    uint32_t more;  // load_pairs: half a word past them, in lane 0
    bool shift;     // load_pairs: the words still start one column early (settle)
};
__device__ __forceinline__ void ld_v8(const void* p, uint32_t* w) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void st_v8(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
template <typename T>
__device__ __forceinline__ T get(const Raw<T>& a, int j) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(a.w[j]);
    } else {
        const unsigned short u = (unsigned short)(a.w[j >> 1] >> (16 * (j & 1)));
        return *reinterpret_cast<const T*>(&u);
    }
}
// Even values first: of two that share a word, the even one clears it.
template <typename T>
__device__ __forceinline__ void put(Raw<T>& a, int j, T v) {
    if constexpr (sizeof(T) == 4) {
        a.w[j] = __float_as_uint(v);
    } else {
        const uint32_t u = *reinterpret_cast<const unsigned short*>(&v);
        if (j & 1) a.w[j >> 1] |= u << 16;
        else a.w[j >> 1] = u;
    }
}

// The same two at a time.  These kernels issue an instruction in three cycles of four and more when written value by
// value, so the arithmetic is packed: pairs of f32 in one instruction, sums of 16-bit rows in their own type (an
// exact sum rounded once).
template <typename T>
__device__ __forceinline__ void add_rows(Raw<T>& x, const Raw<T>& r) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; i += 2) {
        if constexpr (sizeof(T) == 4) {
            float lo, hi;
            f2_unpack(add_f32x2(f2_pack(__uint_as_float(x.w[i]), __uint_as_float(x.w[i + 1])),
                                f2_pack(__uint_as_float(r.w[i]), __uint_as_float(r.w[i + 1]))), lo, hi);
            x.w[i] = __float_as_uint(lo);
            x.w[i + 1] = __float_as_uint(hi);
        } else {
            using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
            for (int k = i; k < i + 2; ++k) {
                const T2 s = __hadd2(*reinterpret_cast<const T2*>(&x.w[k]), *reinterpret_cast<const T2*>(&r.w[k]));
                x.w[k] = *reinterpret_cast<const uint32_t*>(&s);
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void widen(const Raw<T>& a, float (&v)[kPer]) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(a.w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a.w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(a.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(a.w[i] & 0xFFFF0000u);
        }
    }
}
__device__ __forceinline__ void scale16(float (&v)[kPer], float s) {
    const uint64_t ss = f2_pack(s, s);
#pragma unroll
    for (int j = 0; j < kPer; j += 2) f2_unpack(mul_f32x2(f2_pack(v[j], v[j + 1]), ss), v[j], v[j + 1]);
}

// The column of value j of a lane in the chunk from c0.
template <bool kVec>
__device__ __forceinline__ int column(int c0, int lane, int j) {
    return kVec ? c0 + lane * kPer + j : c0 + 64 * (j >> 1) + 2 * lane + (j & 1);
}

// The second half of a lane's word and the first of the word after it, which the next lane has, or lane 0 as its next.
__device__ __forceinline__ uint32_t shifted(uint32_t mine, uint32_t lane0_next, int lane) {
    const uint32_t next = __shfl_sync(kAll, lane == 0 ? lane0_next : mine, (lane + 1) & 31);
    return (mine >> 16) | (next << 16);
}

// A lane's pairs of columns of a row of K from anywhere, zeros at and past K; settle() puts them in place (apart, so that
// loads can be under way for long: the shift would wait for them).
template <typename T>
__device__ __forceinline__ void load_pairs(const T* row, int c0, int lane, int K, Raw<T>& a) {
    if constexpr (sizeof(T) == 4) {
        const bool pair = (reinterpret_cast<uintptr_t>(row) & 7u) == 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = column<false>(c0, lane, 2 * i);
            const uint32_t* p = reinterpret_cast<const uint32_t*>(row) + c;
            uint2 u = make_uint2(0, 0);
            if (pair && c + 2 <= K) {
                u = *reinterpret_cast<const uint2*>(p);
            } else {
                if (c < K) u.x = p[0];
                if (c + 1 < K) u.y = p[1];
            }
            a.w[2 * i] = u.x;
            a.w[2 * i + 1] = u.y;
        }
    } else {
        const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
        if ((reinterpret_cast<uintptr_t>(row) & 2u) == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = column<false>(c0, lane, 2 * i);
                a.w[i] = c + 2 <= K ? *reinterpret_cast<const uint32_t*>(r + c) : (c < K ? r[c] : 0u);
            }
        } else {
            // columns c - 1 and c: the ones that share a word
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = column<false>(c0, lane, 2 * i);
                if (c == 0) a.w[i] = (uint32_t)r[0] << 16;
                else a.w[i] = c < K ? *reinterpret_cast<const uint32_t*>(r + c - 1) : (c - 1 < K ? r[c - 1] : 0u);
            }
            a.more = lane == 0 && c0 + kChunk - 1 < K ? r[c0 + kChunk - 1] : 0u;
        }
        a.shift = (reinterpret_cast<uintptr_t>(row) & 2u) != 0;
    }
}
template <typename T, bool kVec>
__device__ __forceinline__ void settle(Raw<T>& a, int lane) {
    if constexpr (!kVec && sizeof(T) == 2) {
        if (!a.shift) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) a.w[i] = shifted(a.w[i], i < 7 ? a.w[i + 1] : a.more, lane);
    }
}
template <typename T>
__device__ __forceinline__ void store_pairs(T* row, int c0, int lane, int K, const Raw<T>& a) {
    if constexpr (sizeof(T) == 4) {
        const bool pair = (reinterpret_cast<uintptr_t>(row) & 7u) == 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = column<false>(c0, lane, 2 * i);
            uint32_t* p = reinterpret_cast<uint32_t*>(row) + c;
            if (pair && c + 2 <= K) {
                *reinterpret_cast<uint2*>(p) = make_uint2(a.w[2 * i], a.w[2 * i + 1]);
            } else {
                if (c < K) p[0] = a.w[2 * i];
                if (c + 1 < K) p[1] = a.w[2 * i + 1];
            }
        }
    } else {
        uint16_t* r = reinterpret_cast<uint16_t*>(row);
        if ((reinterpret_cast<uintptr_t>(row) & 2u) == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = column<false>(c0, lane, 2 * i);
                if (c + 2 <= K) *reinterpret_cast<uint32_t*>(r + c) = a.w[i];
                else if (c < K) r[c] = (uint16_t)a.w[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = column<false>(c0, lane, 2 * i);
                const uint32_t u = shifted(a.w[i], a.w[i < 7 ? i + 1 : i], lane);  // columns c + 1 and c + 2
                if (i == 0 && lane == 0 && c < K) r[c] = (uint16_t)a.w[0];
                if (c + 3 <= K && !(i == 7 && lane == 31)) *reinterpret_cast<uint32_t*>(r + c + 1) = u;
                else if (c + 2 <= K) r[c + 1] = (uint16_t)u;
            }
        }
    }
}

// A lane's sixteen values of a row of K, zeros at and past K.  align: of the row, in bytes (32, 16 or less).
template <typename T, bool kVec>
__device__ __forceinline__ void load16(const T* row, int c0, int lane, int K, int align, Raw<T>& a) {
    constexpr int kW = Raw<T>::kWords;
    if constexpr (!kVec) {
        load_pairs(row, c0, lane, K, a);
    } else if (column<kVec>(c0, lane, kPer) <= K) {
        const T* p = row + column<kVec>(c0, lane, 0);
        if (align >= 32) {
#pragma unroll
            for (int i = 0; i < kW / 8; ++i) ld_v8(reinterpret_cast<const uint32_t*>(p) + 8 * i, a.w + 8 * i);
        } else {
#pragma unroll
            for (int i = 0; i < kW / 4; ++i) {
                const uint4 u = reinterpret_cast<const uint4*>(p)[i];
                a.w[4 * i] = u.x, a.w[4 * i + 1] = u.y, a.w[4 * i + 2] = u.z, a.w[4 * i + 3] = u.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kW; ++i) a.w[i] = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (column<kVec>(c0, lane, j) < K) put(a, j, row[column<kVec>(c0, lane, j)]);
    }
}
template <typename T, bool kVec>
__device__ __forceinline__ void store16(T* row, int c0, int lane, int K, int align, const Raw<T>& a) {
    constexpr int kW = Raw<T>::kWords;
    if constexpr (!kVec) {
        store_pairs(row, c0, lane, K, a);
    } else if (column<kVec>(c0, lane, kPer) <= K) {
        T* p = row + column<kVec>(c0, lane, 0);
        if (align >= 32) {
#pragma unroll
            for (int i = 0; i < kW / 8; ++i) st_v8(reinterpret_cast<uint32_t*>(p) + 8 * i, a.w + 8 * i);
        } else {
#pragma unroll
            for (int i = 0; i < kW / 4; ++i)
                reinterpret_cast<uint4*>(p)[i] = make_uint4(a.w[4 * i], a.w[4 * i + 1], a.w[4 * i + 2], a.w[4 * i + 3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (column<kVec>(c0, lane, j) < K) row[column<kVec>(c0, lane, j)] = get(a, j);
    }
}

// The largest finite magnitude (as bits) of the block of each of a lane's values: kVec: one block a lane, in top[0];
// else block i holds values 4 i .. 4 i + 3 of every lane.  A maximum passes over NaNs; infinities become NaN in v.
template <bool kVec>
__device__ __forceinline__ void block_tops(float (&v)[kPer], uint32_t (&top)[4]) {
    constexpr int kBlocks = kVec ? 1 : 4, kIn = kPer / kBlocks;
    uint32_t most = 0;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        float t = fmaxf(fabsf(v[b * kIn]), fabsf(v[b * kIn + 1]));
#pragma unroll
        for (int i = 2; i < kIn; i += 2) t = fmax3(t, fabsf(v[b * kIn + i]), fabsf(v[b * kIn + i + 1]));
        t = fmaxf(t, 0.0f);  // all NaN
        top[b] = __float_as_uint(t);
        most = max(most, top[b]);
    }
    if (__any_sync(kAll, most >= kInfBits)) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < kIn; ++i) {
                if (__float_as_uint(fabsf(v[b * kIn + i])) >= kInfBits) v[b * kIn + i] = __uint_as_float(0x7FFFFFFFu);
                else t = fmaxf(t, fabsf(v[b * kIn + i]));
            }
            top[b] = __float_as_uint(t);
        }
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        if constexpr (kVec) {
#pragma unroll
            for (int s = 4; s; s >>= 1) top[b] = max(top[b], __shfl_xor_sync(kAll, top[b], s));
        } else {
            top[b] = __reduce_max_sync(kAll, top[b]);
        }
    }
}

// A value within kNear steps of f32 of the middle between two (normal) codes, where its last bits decide, gives at most
// kMiddle: the 20 fraction bits that a code drops, around one half, shifted up by 12.  Four steps of 2^-24 (where a
// significand is near 2): the norm's values carry the roundings of 1 / sqrt and of two products, half a step each, and
// half of the mean's error; a wider window finds no more.
constexpr uint32_t kNear = 4, kMiddle = 2 * kNear << 12;
__device__ __forceinline__ uint32_t middle(float v) { return (__float_as_uint(v) << 12) + ((kNear - 0x80000u) << 12); }

// 512 columns of a row from c0, sixteen values to a lane (zeros past K), into codes and scale bytes.  All lanes take
// part.  kAgain: the values have been rounded to f32, and a code of one near a middle may be the wrong neighbour;
// returns which of the lane's values are (bit j), and the scale bytes.
template <bool kVec, bool kAgain>
__device__ __forceinline__ uint32_t encode16(float (&v)[kPer], const Fp8Rows& o, long long row, int c0, int lane, uint32_t& word) {
    uint32_t top[4];
    block_tops<kVec>(v, top);
    uint8_t* codes = o.codes + row * o.row_bytes;
    if constexpr (kVec) {
        const uint32_t byte = fp8_scale_byte(top[0]);
        word = __reduce_or_sync(kAll, byte << (8 * (lane >> 3)));
        scale16(v, fp8_scale_inverse(byte));  // by a power of two: exact
        const int c = column<kVec>(c0, lane, 0);
        if (c < o.K)  // rows are K rounded up to 16 bytes long at least
            *reinterpret_cast<uint4*>(codes + c) =
                make_uint4(fp8_pack4(v[0], v[1], v[2], v[3]), fp8_pack4(v[4], v[5], v[6], v[7]),
                           fp8_pack4(v[8], v[9], v[10], v[11]), fp8_pack4(v[12], v[13], v[14], v[15]));
    } else {
        word = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t byte = fp8_scale_byte(top[b]);
            word |= byte << (8 * b);
            const float inv = fp8_scale_inverse(byte);
#pragma unroll
            for (int i = 4 * b; i < 4 * b + 4; ++i) v[i] *= inv;
            const uint32_t u = fp8_pack4(v[4 * b], v[4 * b + 1], v[4 * b + 2], v[4 * b + 3]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = column<kVec>(c0, lane, 4 * b + 2 * i);
                if (c < o.Kp) *reinterpret_cast<uint16_t*>(codes + c) = (uint16_t)(u >> (16 * i));
            }
        }
    }
    uint8_t* s = o.scales + fp8_scale_offset(row, c0 >> 7, o.ktiles);
    if (c0 + 3 * 128 < o.K) {
        if (lane == 0) *reinterpret_cast<uint32_t*>(s) = word;
    } else if (lane < 4 && c0 + lane * 128 < o.K) {  // bytes of blocks past K stay as they were
        s[lane] = (uint8_t)(word >> (8 * lane));
    }
    uint32_t near = 0;
    if constexpr (kAgain) {
        uint32_t least = middle(v[0]);
#pragma unroll
        for (int j = 1; j + 1 < kPer; j += 2) least = __vimin3_u32(least, middle(v[j]), middle(v[j + 1]));
        if (min(least, middle(v[kPer - 1])) <= kMiddle) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) near |= middle(v[j]) <= kMiddle ? 1u << j : 0u;
        }
    }
    return near;
}

// (row, 512-column chunk) of a warp's unit; 32-bit arithmetic where the units allow it.
__device__ __forceinline__ void unit_at(long long unit, int ktiles, bool narrow, long long& row, int& chunk) {
    if (narrow) {
        const uint32_t u = (uint32_t)unit, r = u / (uint32_t)ktiles;
        row = r;
        chunk = (int)(u - r * (uint32_t)ktiles);
    } else {
        row = unit / ktiles;
        chunk = (int)(unit % ktiles);
    }
}
// The start of token row m, L tokens to a sequence unless rows are evenly spaced.
template <typename P>
__device__ __forceinline__ P* row_at(P* base, long long m, bool even, long long L, long long nb1, long long nb2) {
    using Bytes = typename std::conditional<std::is_const<P>::value, const char, char>::type;
    Bytes* b = reinterpret_cast<Bytes*>(base);
    return reinterpret_cast<P*>(even ? b + m * nb1 : b + (m / L) * nb2 + (m % L) * nb1);
}

// Threads of the norm that an SM is to hold in CTAs of at most 256 (4,096 columns): 768 (80 registers) for 16-bit rows,
// whose loads in flight are small, 512 (128 registers) for f32.  31,744 x 4,096 bf16 with residual, before its arithmetic
// was packed (136 us since): 512 threads 176 us, 768 154 us, 1,024 170 us (spills).  CTAs for wider rows are bounded by
// their own size, one to an SM: of 288 to 512 threads with 103 registers and more, above 8,192 columns of 544 to 1,024 with
// 64, which spill.  (16,384 x 5,120 bf16 with residual 156.5 us; with two CTAs an SM in the grid, the second of which
// waits for the first, 157.9.)
template <typename T>
__host__ __device__ constexpr int norm_threads() { return sizeof(T) == 2 ? 768 : 512; }
// CTAs of `most` threads that the registers leave room for.
template <typename T>
__host__ __device__ constexpr int norm_ctas(int most) { return norm_threads<T>() / most > 0 ? norm_threads<T>() / most : 1; }

// The sum over a warp of values >= 0 as total * 2^exponent, to 2^-26 of the largest: in whole numbers, which one
// instruction adds exactly (in f32 the five rounded steps would be off by as much as a value's own rounding, and move
// every value of the row across the middles between codes).  Not finite: an exponent of 1024 + 128, the largest in total.
struct WarpSum {
    uint32_t total;
    int exponent;
    __device__ float value() const {
        if (exponent > 1024) return __uint_as_float(total);
        const int half = exponent >> 1;  // (two factors: one may not be a normal number)
        return (float)total * __uint_as_float((uint32_t)(half + 127) << 23) * __uint_as_float((uint32_t)(exponent - half + 127) << 23);
    }
    __device__ double exact() const {
        if (exponent > 1024) return __uint_as_float(total);
        return (double)total * __hiloint2double((exponent + 1023) << 20, 0);
    }
};
__device__ __forceinline__ WarpSum warp_sum(float v) {
    const uint32_t top = __reduce_max_sync(kAll, __float_as_uint(v) & 0x7FFFFFFFu);
    if (top >= kInfBits) return WarpSum{top, 1024 + 128};
    const bool low = top < 64u << 23;  // lifted, so that the factor below is a normal number
    const float lift = low ? 0x1p64f : 1.0f;
    const uint32_t e = __float_as_uint(__uint_as_float(top) * lift) >> 23;  // lifted values are below 2^(e - 126)
    const float unit = __uint_as_float((279u - e) << 23);                   // 2^(152 - e): below 2^26
    return WarpSum{__reduce_add_sync(kAll, __float2uint_rn(v * lift * unit)), (int)e - 152 - (low ? 64 : 0)};
}

// 1 / sqrt(mean) within about half a step: CUDA's approximation and one Newton step.
__device__ __forceinline__ float inverse_root(float mean) {
    const float y = rsqrtf(mean);
    const float more = fmaf(0.5f * y, fmaf(-mean * y, y, 1.0f), y);
    return mean < __uint_as_float(kInfBits) ? more : y;
}

// The codes of some of a lane's values (bit j of `near`) once more, from h, the gain and the row's squares: |v| is above
// the middle M between its neighbours if (h g f)^2 K > M^2 (squares + K eps), f being one over the block's scale.  The
// comparison is in 64 bits; the squares are what the lanes' f32 chains of sixteen gave, in normal values off by 2^-25 (64
// columns) to 2^-28 (4,096) of their sum, and never by more than 2^-19.  So codes are the exact value's where the squares
// have an exact f32 sum, and elsewhere but for 1e-7 of all (without this 5.4e-7; elementary f32 operations 5.7e-7 to
// 7.1e-7).  One value in 115,000 comes here.  It costs the f32 norm of 31,744 x 1,792 89 -> 100 us with its read-back and
// the bf16 norm of 4,096 columns 196 -> 201 us: the first visits on an SM fetch instructions that the rows streaming
// through L2 have pushed out (a visit that does nothing but store a byte takes 93 us).
template <typename T, bool kVec>
__device__ __forceinline__ void encode_again(const Norm8Params& p, long long m, int c0, int lane, uint32_t near, uint32_t word,
                                             const Raw<T>& rows, const float (&gain)[kPer], float inv, double squares) {
    const double right = fma((double)p.out.K, (double)p.eps, squares);
    for (; near; near &= near - 1) {
        const int j = __ffs(near) - 1, c = column<kVec>(c0, lane, j);
        if (c >= p.out.K) break;
        float h = 0.0f, g = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (i == j) h = to_f32(get(rows, i)), g = gain[i];
        const float f = fp8_scale_inverse(word >> (8 * (kVec ? lane >> 3 : j >> 2)) & 255u);
        const uint32_t about = __float_as_uint(h * inv * g * f);
        const uint32_t middle = (about & 0xFFF00000u) | 0x80000u;
        const double a = (double)h * g * f, b = __uint_as_float(middle);
        const double left = a * a * p.out.K, bar = b * b * right;
        // one step of f32 to the side of the value (magnitudes: the sign is the top bit)
        const uint32_t bits = left > bar ? middle + 1 : (left < bar ? middle - 1 : middle);
        p.out.codes[m * p.out.row_bytes + c] = (uint8_t)fp8_pack4(__uint_as_float(bits), 0.0f, 0.0f, 0.0f);
    }
}

// One row at a time by the CTA (kWarpRows: by each warp of its own), a warp holding one chunk of 512 columns, or two
// in CTAs of more than 512 threads.  The CTA stays and takes every gridDim.x-th row: the gain is read once, and
// the next row is on its way (in registers) while this one is summed, divided and written.  One pass over the data.
template <typename T, bool kVec, int kMaxThreads, bool kWarpRows>
__global__ void __launch_bounds__(kMaxThreads, norm_ctas<T>(kMaxThreads)) norm8_kernel(const __grid_constant__ Norm8Params p) {
    constexpr int kChunks = kMaxThreads > 512 ? 2 : 1;
    constexpr bool kAhead = kChunks == 1;  // a second row of 32 columns a thread does not fit the registers
    __shared__ WarpSum part[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int K = p.out.K;
    launch_next();
    wait_for_previous();
    const int c0 = kWarpRows ? 0 : warp * (kChunks * kChunk);
    const long long first = kWarpRows ? (long long)blockIdx.x * warps + warp : blockIdx.x;
    const long long step = kWarpRows ? (long long)gridDim.x * warps : gridDim.x;
    const long long rows = p.out.rows;
    float g[kChunks][kPer];
#pragma unroll
    for (int q = 0; q < kChunks; ++q) {
        Raw<float> a;
        if (p.gain && kAhead) load16<float, kVec>(p.gain, c0 + q * kChunk, lane, K, p.gain_align, a);
#pragma unroll
        for (int j = 0; j < kPer; ++j) g[q][j] = p.gain && kAhead ? __uint_as_float(a.w[j]) : 1.0f;
    }
    const bool even = p.L >= rows;
    auto fetch = [&](long long m, Raw<T> (&x)[kChunks], Raw<T> (&r)[kChunks]) {
        const T* px = row_at(static_cast<const T*>(p.x), m, even, p.L, p.x_nb1, p.x_nb2);
        const T* pr = row_at(static_cast<const T*>(p.r), m, even, p.L, p.r_nb1, p.r_nb2);
#pragma unroll
        for (int q = 0; q < kChunks; ++q) {
            load16<T, kVec>(px, c0 + q * kChunk, lane, K, p.align, x[q]);
            if (p.r) load16<T, kVec>(pr, c0 + q * kChunk, lane, K, p.align, r[q]);
        }
    };
    Raw<T> x[kChunks], r[kChunks];
    if (kAhead && first < rows) fetch(first, x, r);
    int turn = 0;
    for (long long m = first; m < rows; m += step, turn ^= 1) {
        if (!kAhead) fetch(m, x, r);
        float v[kChunks][kPer];
        Raw<T> s[kChunks];
        uint64_t sums = f2_pack(0.0f, 0.0f);
#pragma unroll
        for (int q = 0; q < kChunks; ++q) {
            settle<T, kVec>(x[q], lane);
            if (p.r) settle<T, kVec>(r[q], lane);
            // the sum is rounded to the rows' type, as it is stored, and the norm is of the stored value
            if (p.r) add_rows(x[q], r[q]);
            if (p.h)
                store16<T, kVec>(row_at(static_cast<T*>(p.h), m, even, p.L, p.h_nb1, p.h_nb2), c0 + q * kChunk, lane, K, p.align,
                                 x[q]);
            s[q] = x[q];
            widen(x[q], v[q]);
#pragma unroll
            for (int j = 0; j < kPer; j += 2) {
                const uint64_t a = f2_pack(v[q][j], v[q][j + 1]);
                sums = fma_f32x2(a, a, sums);
            }
        }
        if (kAhead && m + step < rows) fetch(m + step, x, r);
        float lo, hi;
        f2_unpack(sums, lo, hi);
        const WarpSum mine = warp_sum(lo + hi);
        float sum = mine.value();
        if (!kWarpRows && warps > 1) {
            // two buffers in turn: a warp may be one row ahead of another's reads, not two
            if (lane == 0) part[turn][warp] = mine;
            __syncthreads();
            const int w = lane & ((1 << (32 - __clz(warps - 1))) - 1);  // the warps' sums, over and over along the lanes
            sum = w < warps ? part[turn][w].value() : 0.0f;
#pragma unroll
            for (int s = 16; s; s >>= 1)
                if (s < warps) sum += __shfl_xor_sync(kAll, sum, s);
        }
        const float inv = inverse_root(fmaf(sum, p.inv_cols, p.eps));
#pragma unroll
        for (int q = 0; q < kChunks; ++q) {
            if (!kAhead && p.gain) {
                Raw<float> a;
                load16<float, kVec>(p.gain, c0 + q * kChunk, lane, K, p.gain_align, a);
#pragma unroll
                for (int j = 0; j < kPer; ++j) g[q][j] = __uint_as_float(a.w[j]);
            }
            scale16(v[q], inv);
#pragma unroll
            for (int j = 0; j < kPer; j += 2)
                f2_unpack(mul_f32x2(f2_pack(v[q][j], v[q][j + 1]), f2_pack(g[q][j], g[q][j + 1])), v[q][j], v[q][j + 1]);
            if (c0 + q * kChunk < K) {
                uint32_t word;
                const uint32_t near = encode16<kVec, true>(v[q], p.out, m, c0 + q * kChunk, lane, word);
                if (near) {
                    double squares = mine.exact();
                    if (!kWarpRows && warps > 1) {
                        squares = 0.0;
                        for (int w = 0; w < warps; ++w) squares += part[turn][w].exact();
                    }
                    encode_again<T, kVec>(p, m, c0 + q * kChunk, lane, near, word, s[q], g[q], inv, squares);
                }
            }
        }
    }
}

constexpr int kUnitThreads = 256;  // eight units of a warp each

template <typename T, bool kVec>
__global__ void __launch_bounds__(kUnitThreads) quant8_kernel(const Quant8Params p) {
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * (kUnitThreads / 32) + (threadIdx.x >> 5);
    const long long units = p.out.rows * p.out.ktiles;
    launch_next();
    wait_for_previous();
    if (unit >= units) return;
    long long row;
    int chunk;
    unit_at(unit, p.out.ktiles, units <= 0xffffffffll, row, chunk);
    Raw<T> a;
    load16<T, kVec>(row_at(static_cast<const T*>(p.x), row, p.L >= p.out.rows, p.L, p.x_nb1, p.x_nb2), chunk * kChunk, lane, p.out.K,
                    p.align, a);
    settle<T, kVec>(a, lane);
    float v[kPer];
    widen(a, v);
    uint32_t word;
    encode16<kVec, false>(v, p.out, row, chunk * kChunk, lane, word);
}

// Weight rows of 32-element ggml blocks (q8_0: f16 scale d and 32 int8; q4_0: f16 scale d and 16 bytes, element j in the
// low nibble, j + 16 in the high one, less 8): a lane per ggml block, four to a block of 128, 1,024 columns a warp.
// Blocks are 34 or 18 bytes long, so a lane reads 16-bit words.  (Bringing the warp's bytes into shared memory in
// 16-byte loads first was slower, 13.6 us against 11.0 for 4,096 x 4,096 q8_0: instructions bound it.)  So the codes q
// become f32 by their place in a significand, the largest is found among them, and d and the new scale, a power of
// two, are multiplied once: d * q * 2^-e is exact whichever comes first (11 and 8 significant bits).  Only where the largest
// code is not 0, which bounds |d| by the new scale; a ggml block of zeros under any finite d takes the factor 0.
constexpr int kGgmlWarps = 4;
template <bool kQ4>
__global__ void __launch_bounds__(32 * kGgmlWarps) quant8_ggml_kernel(const uint8_t* w, long long row_bytes, const Fp8Rows o) {
    constexpr int kBytes = kQ4 ? 18 : 34;
    constexpr float kBias = 8388608.0f + (kQ4 ? 8.0f : 128.0f);  // 2^23, and what the codes are raised by
    const int lane = threadIdx.x & 31;
    const int chunks = (o.K + 1023) >> 10;
    const long long unit = (long long)blockIdx.x * kGgmlWarps + (threadIdx.x >> 5), units = o.rows * chunks;
    launch_next();
    wait_for_previous();
    if (unit >= units) return;
    long long row;
    int chunk;
    unit_at(unit, chunks, units <= 0xffffffffll, row, chunk);
    const int c = chunk * 1024 + lane * 32;
    const bool live = c < o.K;  // (K is a multiple of 32: a ggml block is wholly inside)
    const uint16_t* b = reinterpret_cast<const uint16_t*>(w + row * row_bytes + (long long)(live ? c >> 5 : 0) * kBytes);
    float d = live ? __half2float(__ushort_as_half(b[0])) : 0.0f;
    float q[32];
#pragma unroll
    for (int j = 0; j < (kQ4 ? 8 : 16); ++j) {
        const uint32_t u = live ? b[1 + j] : 0u;
        if constexpr (kQ4) {
            q[2 * j] = __uint_as_float(0x4B000000u | (u & 15u)) - kBias;
            q[2 * j + 16] = __uint_as_float(0x4B000000u | (u >> 4 & 15u)) - kBias;
            q[2 * j + 1] = __uint_as_float(0x4B000000u | (u >> 8 & 15u)) - kBias;
            q[2 * j + 17] = __uint_as_float(0x4B000000u | (u >> 12)) - kBias;
        } else {
            const uint32_t r = u ^ 0x8080u;
            q[2 * j] = __uint_as_float(__byte_perm(r, 0x4B000000u, 0x7650)) - kBias;
            q[2 * j + 1] = __uint_as_float(__byte_perm(r, 0x4B000000u, 0x7651)) - kBias;
        }
    }
    float most = fmaxf(fabsf(q[0]), fabsf(q[1]));
#pragma unroll
    for (int j = 2; j < 32; j += 2) most = fmax3(most, fabsf(q[j]), fabsf(q[j + 1]));
    uint32_t top = __float_as_uint(fabsf(d) * most);
    // a ggml block whose scale is not finite is NaN (its zeros too, 0 * d) and does not count
    const bool nan = (__float_as_uint(d) & kInfBits) == kInfBits;
    if (nan) top = 0;
#pragma unroll
    for (int s = 2; s; s >>= 1) top = max(top, __shfl_xor_sync(kAll, top, s));
    const uint32_t byte = fp8_scale_byte(top);
    if (!live) return;
    d = nan ? __uint_as_float(0x7FFFFFFFu) : (most == 0.0f ? 0.0f : d * fp8_scale_inverse(byte));
    uint4* dst = reinterpret_cast<uint4*>(o.codes + row * o.row_bytes + c);
    const uint64_t dd = f2_pack(d, d);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float* a = q + 16 * i + 4 * j;
            f2_unpack(mul_f32x2(f2_pack(a[0], a[1]), dd), a[0], a[1]);
            f2_unpack(mul_f32x2(f2_pack(a[2], a[3]), dd), a[2], a[3]);
            u[j] = fp8_pack4(a[0], a[1], a[2], a[3]);
        }
        dst[i] = make_uint4(u[0], u[1], u[2], u[3]);
    }
    if ((lane & 3) == 0) o.scales[fp8_scale_offset(row, c >> 7, o.ktiles)] = (uint8_t)byte;
}

// Two units a warp: their loads are under way together.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kUnitThreads) dequant8_kernel(const Dequant8Params p) {
    constexpr int kUnits = 2, kWarps = kUnitThreads / 32;
    const int lane = threadIdx.x & 31;
    const long long units = p.in.rows * p.in.ktiles;
    const bool narrow = units <= 0xffffffffll;
    launch_next();
    wait_for_previous();
    long long row[kUnits];
    int c0[kUnits];
    uint32_t codes[kUnits][4], word[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const long long unit = (long long)blockIdx.x * (kWarps * kUnits) + u * kWarps + (threadIdx.x >> 5);
        row[u] = -1;
        if (unit >= units) continue;
        int chunk;
        unit_at(unit, p.in.ktiles, narrow, row[u], chunk);
        c0[u] = chunk * kChunk;
        const uint8_t* src = p.in.codes + row[u] * p.in.row_bytes;
        word[u] = *reinterpret_cast<const uint32_t*>(p.in.scales + fp8_scale_offset(row[u], c0[u] >> 7, p.in.ktiles));
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[u][i] = 0;
        if constexpr (kVec) {
            if (column<kVec>(c0[u], lane, 0) < p.in.K) {  // (a code row is K rounded up to 16 bytes at least)
                const uint4 q = *reinterpret_cast<const uint4*>(src + column<kVec>(c0[u], lane, 0));
                codes[u][0] = q.x, codes[u][1] = q.y, codes[u][2] = q.z, codes[u][3] = q.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < kPer; j += 2)
                if (column<kVec>(c0[u], lane, j) < p.in.K)
                    codes[u][j >> 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(src + column<kVec>(c0[u], lane, j)) << (8 * (j & 2));
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        if (row[u] < 0) continue;
        Raw<T> a;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float s = fp8_scale_value((word[u] >> (8 * (kVec ? lane >> 3 : i))) & 255u);
            float v[4];
            fp8_unpack4(codes[u][i], v);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                f2_unpack(mul_f32x2(f2_pack(v[j], v[j + 1]), f2_pack(s, s)), v[j], v[j + 1]);
                if constexpr (sizeof(T) == 4) {
                    a.w[4 * i + j] = __float_as_uint(v[j]);
                    a.w[4 * i + j + 1] = __float_as_uint(v[j + 1]);
                } else {
                    a.w[2 * i + (j >> 1)] = Pack2<T>::pack(v[j], v[j + 1]);
                }
            }
        }
        store16<T, kVec>(row_at(static_cast<T*>(p.y), row[u], p.L >= p.in.rows, p.L, p.y_nb1, p.y_nb2), c0[u], lane, p.in.K, p.align, a);
    }
}

// Up to 512 columns a warp has a row of its own; to 8,192 a CTA has a warp for every 512 columns; above, a warp for
// every 1,024.  As many CTAs as the GPU holds at one time, by the launch bounds, stay for all rows.
template <typename T, bool kVec>
cudaError_t norm8_typed(const Norm8Params& p, int num_sms, cudaStream_t st) {
    const int K = p.out.K;
    const int chunk = K <= 16 * kChunk ? kChunk : 2 * kChunk;
    const int threads = K <= kChunk ? 128 : (K + chunk - 1) / chunk * 32;
    const int most = K <= kChunk ? 128 : (K <= 8 * kChunk ? 256 : (K <= 16 * kChunk ? 512 : 1024));
    auto kern = most == 128   ? norm8_kernel<T, kVec, 128, true>
                : most == 256 ? norm8_kernel<T, kVec, 256, false>
                : most == 512 ? norm8_kernel<T, kVec, 512, false>
                              : norm8_kernel<T, kVec, 1024, false>;
    const long long per_cta = K <= kChunk ? 4 : 1;
    const long long want = (p.out.rows + per_cta - 1) / per_cta;
    const long long fit = (long long)num_sms * (most * norm_ctas<T>(most) / threads);
    return launch_following(kern, dim3((unsigned)std::min(want, fit)), (unsigned)threads, 0, 1, st, p);
}

unsigned unit_grid(long long units, int per_cta) { return (unsigned)((units + per_cta - 1) / per_cta); }

}  // namespace

cudaError_t launch_norm8(int type, const Norm8Params& p, int num_sms, cudaStream_t st) {
    if (p.out.rows == 0) return cudaSuccess;
    if (p.align >= 16)
        return type == 0 ? norm8_typed<float, true>(p, num_sms, st)
                         : (type == 1 ? norm8_typed<__half, true>(p, num_sms, st) : norm8_typed<__nv_bfloat16, true>(p, num_sms, st));
    return type == 0 ? norm8_typed<float, false>(p, num_sms, st)
                     : (type == 1 ? norm8_typed<__half, false>(p, num_sms, st) : norm8_typed<__nv_bfloat16, false>(p, num_sms, st));
}

cudaError_t launch_quant8(int type, const Quant8Params& p, cudaStream_t st) {
    if (p.out.rows == 0) return cudaSuccess;
    const bool vec = p.align >= 16;
    auto kern = type == 0 ? (vec ? quant8_kernel<float, true> : quant8_kernel<float, false>)
                          : (type == 1 ? (vec ? quant8_kernel<__half, true> : quant8_kernel<__half, false>)
                                       : (vec ? quant8_kernel<__nv_bfloat16, true> : quant8_kernel<__nv_bfloat16, false>));
    return launch_following(kern, dim3(unit_grid(p.out.rows * p.out.ktiles, kUnitThreads / 32)), kUnitThreads, 0, 1, st, p);
}

cudaError_t launch_quant8_ggml(const void* w, bool q4, long long row_bytes, const Fp8Rows& out, cudaStream_t st) {
    if (out.rows == 0) return cudaSuccess;
    return launch_following(q4 ? quant8_ggml_kernel<true> : quant8_ggml_kernel<false>,
                            dim3(unit_grid(out.rows * ((out.K + 1023) / 1024), kGgmlWarps)), 32 * kGgmlWarps, 0, 1, st,
                            static_cast<const uint8_t*>(w), row_bytes, out);
}

cudaError_t launch_dequant8(int type, const Dequant8Params& p, cudaStream_t st) {
    if (p.in.rows == 0) return cudaSuccess;
    const bool vec = p.align >= 16;
    auto kern = type == 0 ? (vec ? dequant8_kernel<float, true> : dequant8_kernel<float, false>)
                          : (type == 1 ? (vec ? dequant8_kernel<__half, true> : dequant8_kernel<__half, false>)
                                       : (vec ? dequant8_kernel<__nv_bfloat16, true> : dequant8_kernel<__nv_bfloat16, false>));
    return launch_following(kern, dim3(unit_grid(p.in.rows * p.in.ktiles, 2 * kUnitThreads / 32)), kUnitThreads, 0, 1, st, p);
}

}  // namespace kd
