// gqa_q8_append.hip -- new K and V rows into the blocks of an 8-bit pool: K rotated at its
// position in double and rounded to f32, then both quantised with the scale of their block.
//
// The rows that one call puts into one (block, KV head) form a run: their largest magnitude a
// gives the smallest power of two s' with s' * qmax >= a (at least 2^-126).  Where the run
// starts at the block's row 0 that is the block's scale; else the block keeps the larger of s'
// and its own, and where it grows the rows before the run move to it.  Powers of two make that
// move an exponent's: an e4m3 code keeps its significand (what falls under its smallest normal
// number aside), an int8 code loses less than one quantum over all of its moves together.
//
// One workgroup of 16 row groups (16 lanes each, 8 dims of a row per lane) takes the runs that
// begin in its window of 16 consecutive tokens, for kHeads KV heads: a run has at most 16 rows, so
// it reads at most 15 rows past the window, and every row is read once.  Skipped tokens end no
// run: they are looked past, in both directions.  The angles of a token's 64 pairs are formed once
// for the kHeads heads.
#include "gqa_device.h"
#include "gqa_internal.h"
#include "gqa_q8.h"

namespace gqa {

namespace {

constexpr int kApWin = 16;                 // tokens of a window
constexpr int kApRows = 2 * kApWin;        // rows a workgroup may read: the window's, and what ends its last run

// The smallest power of two s with s * qmax >= a, at least 2^-126 (a finite, >= 0).  qmax is
// 127 = 1.984375 * 2^6 or 448 = 1.75 * 2^8: the exponent follows from a's bits.
template <int kFmt>
__device__ __forceinline__ float scale_for(float a) {
    constexpr int kExp = kFmt == kQ8E4m3 ? 8 : 6;
    constexpr uint32_t kMant = kFmt == kQ8E4m3 ? 0x600000u : 0x7e0000u;
    const uint32_t u = __float_as_uint(a);
    const int e = static_cast<int>(u >> 23) - kExp + ((u & 0x7fffffu) > kMant ? 1 : 0);
    return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}

// Four values in code units -> four codes, to nearest even, saturating.  NaN: e4m3's NaN, and 0
// for int8, which has none.
template <int kFmt>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4]) {
    if constexpr (kFmt == kQ8E4m3) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = fminf(fmaxf(x[j], -448.0f), 448.0f);
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
        uint32_t r = static_cast<uint32_t>(w);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (x[j] != x[j]) r |= 0x7fu << (8 * j);
        return r;
    } else {
        uint32_t r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float y = x[j] == x[j] ? fminf(fmaxf(rintf(x[j]), -127.0f), 127.0f) : 0.0f;
            r |= (static_cast<uint32_t>(static_cast<int>(y)) & 0xffu) << (8 * j);
        }
        return r;
    }
}

template <int kFmt>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
    if constexpr (kFmt == kQ8E4m3) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
        const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
        x[0] = a[0];
        x[1] = a[1];
        x[2] = b[0];
        x[3] = b[1];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = static_cast<float>(static_cast<int8_t>(w >> (8 * j)));
    }
}

__device__ __forceinline__ float finite_abs(float x) {
    const float y = fabsf(x);
    return y < __builtin_inff() ? y : 0.0f;        // (NaN compares false)
}

// x / s: by the exact inverse where s is a power of two (every scale that an append wrote is).
__device__ __forceinline__ float over_scale(float x, float s, float inv, bool pow2) { return pow2 ? x * inv : x / s; }

}  // namespace

template <int kFmt, int kHeads>
__global__ __launch_bounds__(256) void q8_append_kernel(Q8AppendArgs a) {
    __shared__ int32_t s_slot[kApRows], s_tok[kApRows];
    __shared__ int32_t s_lead[kApRows];                        // row that leads the run, -1: not this workgroup's
    __shared__ float s_max[2][kHeads][kApRows];                // largest magnitude of each row: K, V
    __shared__ float s_old[2][kHeads][kApWin];                 // scale of the block that a run leads into
    const int tid = threadIdx.x, lane = tid & 15, group = tid >> 4;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kApWin;
    const int h0 = blockIdx.y * kHeads;

    // The rows' slots and runs: a row leads where the valid one before it lies in another block.
    if (tid < kWave) {
        const int64_t slots_end = static_cast<int64_t>(a.pool.n_blocks) * kQ8Block;
        auto slot_of = [&](int64_t t) {
            const int32_t slot = t >= 0 && t < a.n_tokens ? a.slots[t] : -1;
            return slot >= 0 && slot < slots_end ? slot : -1;
        };
        // Lanes 0 .. 15: the window; 16 .. 31: the tokens before it.
        const int32_t slot = tid < 2 * kApWin ? slot_of(tid < kApWin ? t0 + tid : t0 + tid - 2 * kApWin) : -1;
        const uint64_t valid = __ballot(slot >= 0);
        const uint32_t in = static_cast<uint32_t>(valid) & 0xffffu;
        int before = -1;                                       // block of the last valid token before the window
        if (in) {
            const uint32_t prev = static_cast<uint32_t>(valid >> kApWin);
            if (prev) before = __shfl(slot, kApWin + 31 - __clz(prev)) >> 4;
            for (int64_t t = t0 - kApWin; !prev && before < 0 && t > 0; t -= kWave) {
                const int32_t s = slot_of(t - kWave + tid);
                const uint64_t v = __ballot(s >= 0);
                if (v) before = __shfl(s, 63 - __clzll(v)) >> 4;
            }
        }
        const uint32_t below = in & ((1u << (tid & 15)) - 1);  // valid tokens of the window before this one
        const int left = __shfl(slot, below ? 31 - __clz(below) : 0) >> 4;
        const bool lead = tid < kApWin && slot >= 0 && (slot >> 4) != (below ? left : before);
        const uint32_t leads = static_cast<uint32_t>(__ballot(lead));
        const uint32_t upto = leads & ((2u << (tid & 15)) - 1);
        if (tid < kApWin) {
            s_slot[tid] = slot;
            s_tok[tid] = static_cast<int32_t>(t0) + tid;
            s_lead[tid] = slot >= 0 && upto ? 31 - __clz(upto) : -1;
            s_lead[kApWin + tid] = -1;
        }
        // What the window's last run has behind it.
        if (leads) {
            const int32_t run = __shfl(slot, 31 - __clz(in)) >> 4;
            int got = 0;
            for (int64_t t = t0 + kApWin; t < a.n_tokens && got < kApWin; t += kWave) {
                const int32_t s = slot_of(t + tid);
                const uint64_t stop = __ballot(s >= 0 && (s >> 4) != run);
                uint64_t more = __ballot(s >= 0);
                if (stop) more &= (stop & -stop) - 1;
                const int at = kApWin + got + __popcll(more & ((1ull << tid) - 1));
                if (((more >> tid) & 1) && at < kApRows) {
                    s_slot[at] = s;
                    s_tok[at] = static_cast<int32_t>(t) + tid;
                    s_lead[at] = 31 - __clz(leads);
                }
                got += __popcll(more);
                if (stop) break;
            }
        }
    }
    __syncthreads();

    // Read and rotate; each row's largest magnitude.
    float x[2][2][kHeads][8];                                  // [row round][K, V]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = group + r * kApWin;
        if (s_lead[row] < 0) continue;
        const int64_t t = s_tok[row];
        uint2 w[2][kHeads][2];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const uint16_t* kr = a.k_new + t * a.k_token_stride + (h0 + h) * kD + 4 * lane;
            const uint16_t* vr = a.v_new + t * a.v_token_stride + (h0 + h) * kD + 4 * lane;
            w[0][h][0] = *reinterpret_cast<const uint2*>(kr);
            w[0][h][1] = *reinterpret_cast<const uint2*>(kr + kPairs);
            w[1][h][0] = *reinterpret_cast<const uint2*>(vr);
            w[1][h][1] = *reinterpret_cast<const uint2*>(vr + kPairs);
        }
        if (r == 0 && s_lead[row] == row && lane < 2 * kHeads) {      // (a lead lies in the first round)
            const float* sc = (lane & 1) ? a.pool.v_scale : a.pool.k_scale;
            const float old = sc[static_cast<int64_t>(s_slot[row] >> 4) * a.pool.scale_block_stride +
                                 (h0 + (lane >> 1)) * a.pool.scale_head_stride];
            s_old[lane & 1][lane >> 1][row] = old > 0.0f && old < __builtin_inff() ? old : 0.0f;
        }
        double sn[4], cs[4];
        if (a.rope) {
            const int64_t pos = a.positions[t];
#pragma unroll
            for (int j = 0; j < 4; ++j) rope_sincos(pos, a.rope_table.inv_freq[4 * lane + j], sn[j], cs[j]);
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                float(&y)[8] = x[r][kv][h];
                y[0] = bf16_lo(w[kv][h][0].x);
                y[1] = bf16_hi(w[kv][h][0].x);
                y[2] = bf16_lo(w[kv][h][0].y);
                y[3] = bf16_hi(w[kv][h][0].y);
                y[4] = bf16_lo(w[kv][h][1].x);
                y[5] = bf16_hi(w[kv][h][1].x);
                y[6] = bf16_lo(w[kv][h][1].y);
                y[7] = bf16_hi(w[kv][h][1].y);
                if (kv == 0 && a.rope) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const double u = y[j], v = y[4 + j];
                        y[j] = static_cast<float>(u * cs[j] - v * sn[j]);
                        y[4 + j] = static_cast<float>(u * sn[j] + v * cs[j]);
                    }
                }
                float m = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(y[j]));
                m = row16_max(m);
                if (lane == 0) s_max[kv][h][row] = m;
            }
        }
    }
    __syncthreads();

    // The run's scale, the codes, and the rows before the run where its block's scale grows.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = group + r * kApWin;
        const int lead = s_lead[row];
        if (lead < 0) continue;
        float m[2][kHeads] = {};
        int first = kQ8Block;                                  // the run's first row in its block
        for (int i = lead; i < kApRows; ++i) {
            if (s_lead[i] != lead) continue;
            first = min(first, s_slot[i] & 15);
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
                m[0][h] = fmaxf(m[0][h], s_max[0][h][i]);
                m[1][h] = fmaxf(m[1][h], s_max[1][h][i]);
            }
        }
        const int64_t blk = s_slot[row] >> 4;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            uint8_t* codes = const_cast<uint8_t*>(kv ? a.pool.v : a.pool.k) + blk * a.pool.block_stride;
            float* scales = const_cast<float*>(kv ? a.pool.v_scale : a.pool.k_scale);
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
                const float old = first > 0 ? s_old[kv][h][lead] : 0.0f;
                const float s = fmaxf(old, scale_for<kFmt>(m[kv][h]));
                const bool pow2 = (__float_as_uint(s) & 0x7fffffu) == 0;
                const float inv = 1.0f / s;
                uint8_t* base = codes + (h0 + h) * a.pool.head_stride + 4 * lane;
                uint8_t* dst = base + (s_slot[row] & 15) * a.pool.pos_stride;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = over_scale(x[r][kv][h][4 * half + j], s, inv, pow2);
                    *reinterpret_cast<uint32_t*>(dst + half * kPairs) = encode4<kFmt>(y);
                }
                if (row != lead) continue;
                if (lane == 0) scales[blk * a.pool.scale_block_stride + (h0 + h) * a.pool.scale_head_stride] = s;
                if (first == 0 || s == old) continue;
                const float ratio = old / s;
                for (int i = 0; i < first; ++i) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t* at = reinterpret_cast<uint32_t*>(base + i * a.pool.pos_stride + half * kPairs);
                        float y[4];
                        decode4<kFmt>(*at, y);
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] *= ratio;
                        *at = encode4<kFmt>(y);
                    }
                }
            }
        }
    }
}

template <int kFmt>
static hipError_t launch_append(const Q8AppendArgs& a, hipStream_t stream) {
    const unsigned windows = static_cast<unsigned>((static_cast<int64_t>(a.n_tokens) + kApWin - 1) / kApWin);
    hipLaunchKernelGGL((q8_append_kernel<kFmt, 1>), dim3(windows, kHkv), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_q8_append(const Q8AppendArgs& a, int format, hipStream_t stream) {
    return format == kQ8E4m3 ? launch_append<kQ8E4m3>(a, stream) : launch_append<kQ8Int8>(a, stream);
}

}  // namespace gqa
