// What the warp-specialised tensor-core kernels share: tile constants, the ring position, giving up, and the host side's
// tensor maps.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace rdb {

constexpr int BM = 128;            // rows of one MMA (TMEM lanes)
constexpr int BK = 64;             // bf16 elements per 128-byte swizzle row
constexpr int UMMA_K = 16;         // K extent of one tcgen05.mma for 16-bit inputs
constexpr int SUB_BYTES = BM * BK * 2;  // one [128 x 64] bf16 sub-tile
constexpr int TMEM_COLS = 512;

struct PipeState {
    uint32_t idx = 0, phase = 0;
    template <int STAGES> __device__ __forceinline__ void advance() {
        if (++idx == STAGES) { idx = 0; phase ^= 1; }
    }
};

__device__ __forceinline__ void raise_abort(volatile int *abort_flag, int32_t *status, int code) {
    *abort_flag = 1;
    if (status) atomicCAS(status, 0, code);
}

// ---- implemented in umma_gemm.cu ----------------------------------------------------------------
// bf16 (or float32) matrix with `inner` contiguous elements per row, `outer` rows, row pitch ld elements.  A row of a box takes the
// swizzle's width in shared memory: boxes are 128 bytes wide, or 64 with the 64-byte swizzle.
int make_tmap(CUtensorMap *m, const void *base, int64_t inner, int64_t outer, int64_t ld, uint32_t box_inner, uint32_t box_outer,
              bool f32 = false, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B);
int max_resident_pairs();          // CTA pairs (one CTA per SM) that can be resident at once
int sm_count();

}  // namespace rdb
