// The C++ host layer's 8-bit path (kd_ops.hpp: Fp8Rows, quantize_fp8, rms_norm_fp8, linear_fp8, dequantize_fp8).
// --cpu: what needs no device.  Otherwise: a norm, a product and the read-back on device 0 against the same steps on
// the host in double, on the values that the 8-bit rows hold.  Prints "OK" or the first failure.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "kd_ops.hpp"

#define CHECK(c)                                       \
    do {                                               \
        if (!(c)) {                                    \
            printf("failed: %s (%d)\n", #c, __LINE__); \
            return 1;                                  \
        }                                              \
    } while (0)

static int cpu() {
    CHECK(kd::Fp8Rows::scale_bytes(4096, 31744) == 248u * 8 * 512);
    CHECK(kd::Fp8Rows::scale_bytes(0, 5) == 0 && kd::Fp8Rows::scale_bytes(128, -1) == 0);
    CHECK(kd::Fp8Rows::suggested_pitch(100) == 128 && kd::Fp8Rows::suggested_pitch(256) == 256);
    kd::Fp8Rows r;
    r.columns = 7;
    r.rows = 3;
    r.pitch = 16;
    const kd_fp8_rows v = r.view();
    CHECK(v.ne[0] == 7 && v.ne[1] == 3 && v.nb1 == 16 && !v.codes && !v.scales);
    kd::Context none(-1, [](kd_attn_log_level, const char*, void*) {}, nullptr);
    kd::Tensor t;
    CHECK(!none.ok() && !kd::ops::quantize_fp8(none, t, r) && !kd::ops::linear_fp8(none, r, r, nullptr, t) &&
          !kd::ops::rms_norm_fp8(none, t, nullptr, nullptr, 1e-6f, nullptr, r) && !kd::ops::dequantize_fp8(none, r, t) &&
          !kd::ops::quantize_fp8(none, kd::Linear{}, r));
    return 0;
}

template <typename T>
static T* device(size_t n) {
    void* p = nullptr;
    return cudaMalloc(&p, n * sizeof(T)) == cudaSuccess ? static_cast<T*>(p) : nullptr;
}
static kd::Fp8Rows rows8(int64_t columns, int64_t rows) {
    kd::Fp8Rows r;
    r.columns = columns;
    r.rows = rows;
    r.pitch = kd::Fp8Rows::suggested_pitch(columns);
    r.codes = device<unsigned char>(r.pitch * (size_t)rows);
    r.scales = device<unsigned char>(kd::Fp8Rows::scale_bytes(columns, rows));
    return r;
}

static int gpu() {
    const int M = 21, K = 200, C = 70;
    kd::Context ctx(0);
    CHECK(ctx.ok());
    std::vector<float> x(M * K), res(M * K), gain(K), w(C * K), bias(C), h(M * K), a(M * K), b(C * K), y(M * C);
    unsigned seed = 1;
    auto next = [&] { return (float)((seed = seed * 1664525u + 1013904223u) >> 8) / 8388608.0f - 1.0f; };
    for (auto* v : {&x, &res, &w, &bias})
        for (auto& f : *v) f = next();
    for (auto& g : gain) g = 1.0f + 0.1f * next();
    float *dx = device<float>(M * K), *dr = device<float>(M * K), *dg = device<float>(K), *dw = device<float>(C * K);
    float *db = device<float>(C), *dh = device<float>(M * K), *da = device<float>(M * K), *dv = device<float>(C * K), *dy = device<float>(M * C);
    CHECK(dx && dr && dg && dw && db && dh && da && dv && dy);
    auto up = [](float* d, const std::vector<float>& v) { return cudaMemcpy(d, v.data(), v.size() * 4, cudaMemcpyHostToDevice) == cudaSuccess; };
    CHECK(up(dx, x) && up(dr, res) && up(dg, gain) && up(dw, w) && up(db, bias));
    auto f32 = [](float* d, int64_t n0, int64_t n1) { return kd::Tensor::contiguous(d, KD_ATTN_TYPE_F32, n0, n1); };
    kd::Tensor tx = f32(dx, K, M), tr = f32(dr, K, M), th = f32(dh, K, M), ta = f32(da, K, M), tv = f32(dv, K, C), ty = f32(dy, C, M);
    const kd::Fp8Rows rx = rows8(K, M), rw = rows8(K, C);
    kd::Linear lin;
    lin.weight = dw;
    lin.type = KD_ATTN_TYPE_F32;
    lin.in_features = K;
    lin.out_features = C;
    lin.nb1 = K * 4;
    CHECK(kd::ops::quantize_fp8(ctx, lin, rw) && kd::ops::rms_norm_fp8(ctx, tx, &tr, dg, 1e-6f, &th, rx));
    CHECK(kd::ops::linear_fp8(ctx, rx, rw, db, ty) && kd::ops::dequantize_fp8(ctx, rx, ta) && kd::ops::dequantize_fp8(ctx, rw, tv));
    CHECK(ctx.device_status());
    auto down = [](std::vector<float>& v, const float* d) { return cudaMemcpy(v.data(), d, v.size() * 4, cudaMemcpyDeviceToHost) == cudaSuccess; };
    CHECK(down(h, dh) && down(a, da) && down(b, dv) && down(y, dy));
    for (int m = 0; m < M; ++m) {
        double sq = 0;
        for (int k = 0; k < K; ++k) {
            CHECK(h[m * K + k] == x[m * K + k] + res[m * K + k]);
            sq += (double)h[m * K + k] * h[m * K + k];
        }
        const double inv = 1.0 / std::sqrt(sq / K + 1e-6);
        for (int k = 0; k < K; ++k) {  // half an e4m3 step: 2^-4 of the value, or 2^-10 of a scale of at most max / 224
            const double v = h[m * K + k] * inv * gain[k];
            CHECK(std::fabs(a[m * K + k] - v) <= std::fabs(v) / 16 + 4.0 / 224 / 1024 + 1e-5);
        }
        for (int c = 0; c < C; ++c) {  // f32 sums of K exact products: K 2^-23 of the sum of magnitudes
            double s = bias[c], room = std::fabs(s);
            for (int k = 0; k < K; ++k) {
                s += (double)a[m * K + k] * b[c * K + k];
                room += std::fabs((double)a[m * K + k] * b[c * K + k]);
            }
            CHECK(std::fabs(y[m * C + c] - s) <= (K + 2) * room / 8388608.0);
        }
    }
    kd::Tensor wrong = f32(dy, C, M - 1);
    CHECK(!kd::ops::linear_fp8(ctx, rx, rw, db, wrong) && !ctx.last_error().empty());
    return 0;
}

int main(int argc, char** argv) {
    const int bad = argc > 1 && !strcmp(argv[1], "--cpu") ? cpu() : gpu();
    if (!bad) printf("OK\n");
    return bad;
}
