// Host-only check: the block-scaled instruction descriptor and the scale-tile descriptor of kd_common.cuh against
// CUTLASS's definitions of the same bit fields (cute::UMMA::make_instr_desc_block_scaled, SmemDescriptor).
// Prints "OK" or the first mismatch.  Built and run by tests/test_fp8_cpu.py.
#include <cstdio>
#include <cute/arch/mma_sm100_desc.hpp>
#include <cute/numeric/numeric_types.hpp>

#include "kd_common.cuh"

using namespace cute;

template <int M, int N>
static int check_idesc() {
    int bad = 0;
    for (uint32_t id = 0; id < 4; ++id) {
        UMMA::InstrDescriptorBlockScaled d =
            UMMA::make_instr_desc_block_scaled<float_e4m3_t, float_e4m3_t, float, float_ue8m0_t, M, N, UMMA::Major::K,
                                               UMMA::Major::K>();
        d.a_sf_id_ = id;
        d.b_sf_id_ = id;
        const uint32_t mine = kd::idesc_e4m3_block(M, N, id);
        if (mine != uint32_t(d)) {
            printf("block-scaled instr desc mismatch M=%d N=%d id=%u mine=%08x cutlass=%08x\n", M, N, id, mine,
                   uint32_t(d));
            ++bad;
        }
    }
    return bad;
}

static int check_scale_tile(uint32_t addr) {
    UMMA::SmemDescriptor d;
    d.desc_ = 0;
    d.version_ = 1;
    d.layout_type_ = uint8_t(UMMA::LayoutType::SWIZZLE_NONE);
    d.start_address_ = uint16_t(addr >> 4);
    d.stride_byte_offset_ = uint16_t(128 >> 4);
    if (kd::desc_scale_tile(addr) != d.desc_) {
        printf("scale tile desc mismatch addr=%u\n", addr);
        return 1;
    }
    return 0;
}

int main() {
    int bad = check_idesc<128, 16>() + check_idesc<128, 80>() + check_idesc<128, 256>() + check_idesc<256, 256>();
    for (uint32_t addr : {0u, 512u, 196608u + 1536u}) bad += check_scale_tile(addr);
    if (!bad) printf("OK\n");
    return bad ? 1 : 0;
}
