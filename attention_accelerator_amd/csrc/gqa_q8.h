// gqa_q8.h -- what the kernels of the 8-bit paged cache share: argument blocks and the two formats'
// conversions.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gqa_device.h"

namespace gqa {

constexpr int kQ8Block = 16;               // positions of a block
constexpr int kQ8Step = 32;                // keys of a step: two blocks
constexpr int kQ8RowB = kD;                // a row's bytes
constexpr int kQ8PlaneB = kQ8Step * kQ8RowB;   // K (or V) of a step in LDS
constexpr int kQ8Int8 = 0;
constexpr int kQ8E4m3 = 1;

struct Q8Pool {
    const uint8_t* k;
    const uint8_t* v;
    const float* k_scale;
    const float* v_scale;
    int64_t block_stride, head_stride, pos_stride;     // bytes
    int64_t scale_block_stride, scale_head_stride;     // floats
    int32_t n_blocks;
};

struct Q8AppendArgs {
    Q8Pool pool;                           // (written through here: the entry point owns the cast)
    const uint16_t* k_new;
    const uint16_t* v_new;
    int64_t k_token_stride, v_token_stride;            // elements
    const int32_t* slots;
    const int32_t* positions;
    int32_t n_tokens;
    int32_t rope;
    RopeTable rope_table;
};

// The sequence that begins in a range and goes on behind it (n = 0: none): its steps there, and a range's.
struct Q8CutSeq {
    int32_t row0, n;
    int64_t left, per;
};

struct Q8AttnArgs {
    Q8Pool pool;
    const uint16_t* q;
    int64_t q_token_stride;                // elements
    const int32_t* block_table;
    const int32_t* seq_len;
    const int32_t* cu;                     // nullptr: one token for each sequence
    uint16_t* out;
    uint32_t* counters;                    // [8][kQ8MaxBatch] pieces written (the heads' far apart: counts in one
                                           // cache line wait for each other); 0 between calls
    Q8CutSeq* cut_seqs;                    // of each range; not of one-token calls
    float* part_o;                         // partial O rows, 128 floats each
    float4* part_ml;                       // (m, M, l, -) of each partial row
    int64_t tile_slot0;                    // first partial row of the tile kernel's part
    int32_t max_blocks;
    int32_t batch;
    int32_t n_tokens;
    int32_t max_new;
    int32_t stream_waves;                  // of the stream kernel: a multiple of 8
    int32_t tile_wgs;                      // workgroups of the tile kernel
    int32_t rope;
    float q_scale;                         // scale * log2(e)
    RopeTable rope_table;
};

struct PagedPlanArgs {
    const int32_t* cached;
    const int32_t* n_new;
    const int32_t* free_blocks;
    const int32_t* n_free;
    int32_t* block_table;
    int64_t table_stride;
    int32_t* seq_len;
    int32_t* cu_new;
    int32_t* slot_map;
    int32_t* positions;
    int32_t* n_free_out;
    int32_t batch;
    int32_t max_blocks;
    int32_t free_capacity;
    int32_t n_rows;
    int32_t rows_per_wg;
};

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t stream);
hipError_t launch_q8_append(const Q8AppendArgs& a, int format, hipStream_t stream);
hipError_t launch_q8_attention(const Q8AttnArgs& a, int format, hipStream_t stream);

constexpr int32_t kQ8MaxBatch = 32768;     // sequences that the counters at a workspace's start are for

// A chunk of more than kQ8StreamMax tokens of one sequence goes to the tile kernel: 16 tokens are the 64
// columns whose sums fit a wave's registers.
constexpr int kQ8StreamMax = 16;
constexpr int kQ8TileTokens = 64;

constexpr int kQ8TileWgsPerCu = 1;         // (eight waves of 256 registers fill a CU)

// Waves of the stream kernel for each CU: one per SIMD.  HBM serves fewer streams at once faster: shuffled
// 2 KB rows copied to LDS by 4, 6 and 8 waves a CU come at 6.85, 6.68 and 6.32 TB/s.  Steps of a wave's
// ring in LDS (8 KB each); a fourth is no faster.
constexpr int kQ8WavesPerCu = 4;
constexpr int kQ8Ring = 3;

// Columns (token, head) of a stream workgroup in tiles of 16: 4 tokens x 4 heads each.
__host__ __device__ constexpr int q8_stream_tiles(int max_new) { return max_new <= 4 ? 1 : max_new <= 8 ? 2 : 4; }

typedef _Float16 q8_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 q8_f16x8 __attribute__((ext_vector_type(8)));
typedef int q8_i32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t q8_u32x4 __attribute__((ext_vector_type(4)));
// LDS pointers keep their address space (32 bits, no generic-pointer checks).
#define GQA_LDS __attribute__((address_space(3)))
typedef GQA_LDS uint8_t q8_lds;

// Two codes of w (bytes 0-1 or 2-3) as fp16: exact for both formats.  int8: the byte with its
// sign bit flipped is the low byte of the fp16 number 1024 + (code + 128).
template <int kFmt, bool kHigh>
__device__ __forceinline__ q8_f16x2 q8_pair(uint32_t w) {
    if constexpr (kFmt == kQ8E4m3) {
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, kHigh);
    } else {
        const uint32_t p = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, kHigh ? 0x04030402u : 0x04010400u);
        return __builtin_bit_cast(q8_f16x2, p) - q8_f16x2{(_Float16)1152.0f, (_Float16)1152.0f};
    }
}

template <int kFmt>
__device__ __forceinline__ q8_f16x8 q8_eight(uint32_t w0, uint32_t w1) {
    const q8_f16x2 a = q8_pair<kFmt, false>(w0), b = q8_pair<kFmt, true>(w0);
    const q8_f16x2 c = q8_pair<kFmt, false>(w1), d = q8_pair<kFmt, true>(w1);
    return q8_f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Values as two fp16, to nearest (v_cvt_pk_f16_f32).
__device__ __forceinline__ q8_f16x2 q8_pack(float lo, float hi) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    return __builtin_convertvector(f32x2_t{lo, hi}, q8_f16x2);
}

}  // namespace gqa
