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
// begin in its window of 16 consecutive tokens.  A run has at most 16 rows, so they are the window's
// and at most 15 behind it, listed in LDS: every row is read once, and where runs follow each
// other without a gap (a prompt's blocks, wherever it starts) a workgroup has 16 of them, a row
// for each group.  Skipped tokens end no run: they are looked past, in both directions.
//
// The workgroup takes its KV heads in turn, the next one's rows requested before this one's are worked
// on; the sines and cosines of a token's 64 pairs, a third of the arithmetic, are formed once.
//
// A small step is one chain of dependent loads (slots; rows, positions, scales) behind a launch: 6 us for
// 64 single tokens, 9 for 24 sequences with 1023 rows.  16384 rows take 39 us, 2.6 TB/s read and
// written, where a copy takes 21: at 160 registers three workgroups share a CU, too few to hide that
// chain (the kernel without its row loads, stores and sines still takes 23 us).
#include "gqa_device.h"
#include "gqa_internal.h"
#include "gqa_q8.h"

namespace gqa {

namespace {

constexpr int kApWin = 16;                 // tokens of a window
constexpr int kApSkip = 8 * kWave;          // skipped tokens passed at a time
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

// Four values in code units -> four codes, to nearest even.
// encode4: any values, saturating; NaN: e4m3's NaN, and 0 for int8, which has none.
// encode4_fit: values that a code is at most half a unit from (what a run's own scale gives).
template <int kFmt>
__device__ __forceinline__ uint32_t encode4(float x0, float x1, float x2, float x3) {
    const float x[4] = {x0, x1, x2, x3};
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
__device__ __forceinline__ uint32_t encode4_fit(const float (&x)[8], int from, float inv) {
    if constexpr (kFmt == kQ8E4m3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[from] * inv, x[from + 1] * inv, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[from + 2] * inv, x[from + 3] * inv, w, true);
        return static_cast<uint32_t>(w);
    } else {
        // 1.5 * 2^23 + n, rounded to nearest even: n's two's complement is in the low bits
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__builtin_fmaf(x[from + j], inv, 12582912.0f));
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u),
                                     0x05040100u);
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

// Eight values over s as codes, dims 4 lane .. and 64 + 4 lane .. of a row.  Where they are finite and s is
// a power of two (every scale that an append wrote is) they are multiplied by its exact inverse and
// fit; the quotients, and the checks for what does not fit, take several times the
// instructions and are left to a branch.
template <int kFmt>
__device__ __forceinline__ void put_codes(uint8_t* dst, const float (&x)[8], float s, bool finite) {
    uint32_t w[2];
    if (__all(finite && (__float_as_uint(s) & 0x7fffffu) == 0)) {
        const float inv = __uint_as_float(0x7f000000u - __float_as_uint(s));       // 2^-e of 2^e
        w[0] = encode4_fit<kFmt>(x, 0, inv);
        w[1] = encode4_fit<kFmt>(x, 4, inv);
    } else {
        w[0] = encode4<kFmt>(x[0] / s, x[1] / s, x[2] / s, x[3] / s);
        w[1] = encode4<kFmt>(x[4] / s, x[5] / s, x[6] / s, x[7] / s);
    }
    *reinterpret_cast<uint32_t*>(dst) = w[0];
    *reinterpret_cast<uint32_t*>(dst + kPairs) = w[1];
}

// The largest magnitude of eight values over the 16 lanes of a row, as bits (as integers they are in
// the magnitudes' order, infinity and NaN above all): `finite` if it is one; if not, what is
// returned is the largest finite one.
__device__ __forceinline__ float row_max(const float (&x)[8], bool& finite) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    const auto over_row = [](uint32_t u) {
        u = max(u, static_cast<uint32_t>(dpp_i<0xB1>(static_cast<int>(u))));
        u = max(u, static_cast<uint32_t>(dpp_i<0x4E>(static_cast<int>(u))));
        u = max(u, static_cast<uint32_t>(dpp_i<0x124>(static_cast<int>(u))));
        return max(u, static_cast<uint32_t>(dpp_i<0x128>(static_cast<int>(u))));
    };
    m = over_row(m);
    finite = m < 0x7f800000u;
    if (!__all(finite)) {
        uint32_t f = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = __float_as_uint(x[j]) & 0x7fffffffu;
            f = max(f, u < 0x7f800000u ? u : 0u);
        }
        m = over_row(f);
    }
    return __uint_as_float(m);
}

}  // namespace

template <int kFmt>
__global__ __launch_bounds__(256) void q8_append_kernel(Q8AppendArgs a, int heads) {
    __shared__ int32_t s_slot[kApRows], s_tok[kApRows];        // the rows of this workgroup's runs
    __shared__ int32_t s_lead[kApRows];                        // the row that leads each one's run
    __shared__ int32_t s_count;
    __shared__ float s_max[2][2][kApRows];                     // [head in turn][K, V] largest magnitude of each row
    __shared__ float s_old[2][2][kApRows];                     // scale of the block that a run leads into
    const int tid = threadIdx.x, lane = tid & 15, group = tid >> 4;
    // (the heads of a window run side by side: a token's heads lie together, and so do a block's)
    const int64_t t0 = static_cast<int64_t>(blockIdx.x / (kHkv / heads)) * kApWin;
    const int h0 = blockIdx.x % (kHkv / heads) * heads;
    double freq[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) freq[j] = a.rope_table.inv_freq[4 * lane + j];

    if (tid < kWave) {
        const int64_t slots_end = static_cast<int64_t>(a.pool.n_blocks) * kQ8Block;
        auto slot_of = [&](int64_t t) {
            const int32_t slot = t >= 0 && t < a.n_tokens ? a.slots[t] : -1;
            return slot >= 0 && slot < slots_end ? slot : -1;
        };
        // Past skipped tokens, eight loads a lane at a time (a padded step may end in thousands of them).
        auto none_of = [&](int64_t t) {
            int32_t top = -1;
#pragma unroll
            for (int j = 0; j < kApSkip / kWave; ++j) top = max(top, slot_of(t + j * kWave + tid));
            return !__any(top >= 0);
        };
        // Lanes 0 .. 15: the window; 16 .. 31: the tokens before it; 32 .. 47: the ones behind.
        const int64_t t_of = tid < kApWin ? t0 + tid : tid < 2 * kApWin ? t0 + tid - 2 * kApWin : t0 + tid - kApWin;
        const int32_t slot = tid < 3 * kApWin ? slot_of(t_of) : -1;
        const uint64_t valid = __ballot(slot >= 0);
        const uint32_t in = static_cast<uint32_t>(valid) & 0xffffu;
        int before = -1;                                       // block of the last valid token before the window
        if (in) {
            const uint32_t prev = static_cast<uint32_t>(valid >> kApWin) & 0xffffu;
            if (prev) before = __shfl(slot, kApWin + 31 - __clz(prev)) >> 4;
            for (int64_t t = t0 - kApWin; !prev && before < 0; t -= kWave) {
                while (t > 0 && none_of(t - kApSkip)) t -= kApSkip;
                if (t <= 0) break;
                const int32_t s = slot_of(t - kWave + tid);
                const uint64_t v = __ballot(s >= 0);
                if (v) before = __shfl(s, 63 - __clzll(v)) >> 4;
            }
        }
        // A row leads where the valid one before it lies in another block; the rows before the first lead
        // are another workgroup's.
        const uint32_t below = in & ((1u << (tid & 15)) - 1);
        const int left = __shfl(slot, below ? 31 - __clz(below) : 0) >> 4;
        const bool lead = tid < kApWin && slot >= 0 && (slot >> 4) != (below ? left : before);
        const uint32_t leads = static_cast<uint32_t>(__ballot(lead));
        int count = 0;
        if (leads) {
            const uint32_t rows = in & ~((1u << __builtin_ctz(leads)) - 1);
            auto listed = [&](int t) { return __popc(rows & ((1u << t) - 1)); };
            if (tid < kApWin && ((rows >> tid) & 1)) {
                const int at = listed(tid);
                s_slot[at] = slot;
                s_tok[at] = static_cast<int32_t>(t0) + tid;
                s_lead[at] = listed(31 - __clz(leads & ((2u << tid) - 1)));
            }
            count = __popc(rows);
            // What the last run has behind the window: among the 16 tokens there, unless some are skipped.
            const int run = __shfl(slot, 31 - __clz(in)) >> 4, of = listed(31 - __clz(leads));
            int32_t s = __shfl(slot, (tid + 2 * kApWin) & (kWave - 1));
            if (tid >= kApWin) s = -1;
            for (int64_t t = t0 + kApWin;;) {
                const uint64_t stop = __ballot(s >= 0 && (s >> 4) != run);
                uint64_t more = __ballot(s >= 0);
                if (stop) more &= (stop & -stop) - 1;
                const int at = count + __popcll(more & ((1ull << tid) - 1));
                if (((more >> tid) & 1) && at < kApRows) {
                    s_slot[at] = s;
                    s_tok[at] = static_cast<int32_t>(t) + tid;
                    s_lead[at] = of;
                }
                count += __popcll(more);
                t += t == t0 + kApWin ? kApWin : kWave;
                if (stop || count >= kApRows) break;
                while (t < a.n_tokens && none_of(t)) t += kApSkip;
                if (t >= a.n_tokens) break;
                s = slot_of(t + tid);
            }
            count = min(count, kApRows);
        }
        if (tid == 0) s_count = count;
    }
    __syncthreads();
    const int count = s_count;
    if (count == 0) return;

    // This group's rows: the listed ones group and group + 16.
    struct Row {
        uint2 w[2][2];                                         // [K, V][dims 4 lane .., 64 + 4 lane ..]
        float old;                                             // lanes 0, 1 of a run's lead: the block's K, V scale
    };
    bool mine[2];
    int lead[2], slot[2];
    double sn[2][4], cs[2][4];
    const uint16_t* src[2][2];
    const float* old_at[2];
    Row row[2];
    auto fetch = [&](int r, int h) {
        Row x;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            x.w[kv][0] = *reinterpret_cast<const uint2*>(src[r][kv] + h * kD);
            x.w[kv][1] = *reinterpret_cast<const uint2*>(src[r][kv] + h * kD + kPairs);
        }
        x.old = old_at[r] ? old_at[r][h * a.pool.scale_head_stride] : 0.0f;
        return x;
    };
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int at = group + r * kApWin;
        mine[r] = at < count;
        if (!mine[r]) continue;
        lead[r] = s_lead[at];
        slot[r] = s_slot[at];
        const int64_t t = s_tok[at];
        src[r][0] = a.k_new + t * a.k_token_stride + 4 * lane;
        src[r][1] = a.v_new + t * a.v_token_stride + 4 * lane;
        // (a run that begins at row 0 has no use for the block's scale)
        old_at[r] = lead[r] == at && lane < 2 && (slot[r] & 15) != 0
                        ? (lane ? a.pool.v_scale : a.pool.k_scale) + static_cast<int64_t>(slot[r] >> 4) * a.pool.scale_block_stride
                        : nullptr;
        row[r] = fetch(r, h0);
        if (a.rope) {
            const int64_t pos = a.positions[t];
#pragma unroll
            for (int j = 0; j < 4; ++j) rope_sincos(pos, freq[j], sn[r][j], cs[r][j]);
        }
    }

    for (int h = h0; h < h0 + heads; ++h) {
        const int turn = h & 1;
        float x[2][2][8];                                      // [row][K, V]
        bool finite[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (!mine[r]) continue;
            const int at = group + r * kApWin;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                float(&y)[8] = x[r][kv];
                const uint2(&w)[2] = row[r].w[kv];
                y[0] = bf16_lo(w[0].x);
                y[1] = bf16_hi(w[0].x);
                y[2] = bf16_lo(w[0].y);
                y[3] = bf16_hi(w[0].y);
                y[4] = bf16_lo(w[1].x);
                y[5] = bf16_hi(w[1].x);
                y[6] = bf16_lo(w[1].y);
                y[7] = bf16_hi(w[1].y);
                if (kv == 0 && a.rope) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const double u = y[j], v = y[4 + j];
                        y[j] = static_cast<float>(u * cs[r][j] - v * sn[r][j]);
                        y[4 + j] = static_cast<float>(u * sn[r][j] + v * cs[r][j]);
                    }
                }
                const float m = row_max(y, finite[r][kv]);
                if (lane == 0) s_max[turn][kv][at] = m;
            }
            const float old = row[r].old;
            if (lead[r] == at && lane < 2) s_old[turn][lane][at] = old > 0.0f && old < __builtin_inff() ? old : 0.0f;
            if (h + 1 < h0 + heads) row[r] = fetch(r, h + 1);
        }
        __syncthreads();                                       // (the other turn's values may be written from here on)

        // The run's scale, the codes, and the rows before the run where its block's scale grows.
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (!mine[r]) continue;
            // The run's largest magnitudes and its first row in the block: a listed row in each lane, twice.
            float m[2] = {}, from_end = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = lane + i * kApWin;
                const bool in_run = at < count && s_lead[at] == lead[r];
                from_end = fmaxf(from_end, in_run ? static_cast<float>(kQ8Block - (s_slot[at] & 15)) : 0.0f);
                m[0] = fmaxf(m[0], in_run ? s_max[turn][0][at] : 0.0f);
                m[1] = fmaxf(m[1], in_run ? s_max[turn][1][at] : 0.0f);
            }
            const int first = kQ8Block - static_cast<int>(row16_max(from_end));
            const int64_t blk = slot[r] >> 4;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const float old = first > 0 ? s_old[turn][kv][lead[r]] : 0.0f;
                const float s = fmaxf(old, scale_for<kFmt>(row16_max(m[kv])));
                uint8_t* base = const_cast<uint8_t*>(kv ? a.pool.v : a.pool.k) + blk * a.pool.block_stride +
                                h * a.pool.head_stride + 4 * lane;
                put_codes<kFmt>(base + (slot[r] & 15) * a.pool.pos_stride, x[r][kv], s, finite[r][kv]);
                if (group + r * kApWin != lead[r]) continue;
                if (lane == 0)
                    const_cast<float*>(kv ? a.pool.v_scale : a.pool.k_scale)[blk * a.pool.scale_block_stride +
                                                                            h * a.pool.scale_head_stride] = s;
                if (first == 0 || s == old) continue;
                const float ratio = old / s;
                for (int i = 0; i < first; ++i) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t* at = reinterpret_cast<uint32_t*>(base + i * a.pool.pos_stride + half * kPairs);
                        float y[4];
                        decode4<kFmt>(*at, y);
                        *at = encode4<kFmt>(y[0] * ratio, y[1] * ratio, y[2] * ratio, y[3] * ratio);
                    }
                }
            }
        }
    }
}

template <int kFmt>
static hipError_t launch_append(const Q8AppendArgs& a, hipStream_t stream) {
    // A workgroup for each window and head while that leaves CUs idle, four heads in turn where there are
    // several rounds of workgroups.  A call in us with 1 and 4 heads in turn: 64 windows 10.4 and 15.2,
    // 1024 windows 60.8 and 43.5 (2 heads: 46.6).
    const int64_t windows = (static_cast<int64_t>(a.n_tokens) + kApWin - 1) / kApWin;
    const int heads = windows * kHkv <= 2048 ? 1 : 4;
    hipLaunchKernelGGL((q8_append_kernel<kFmt>), dim3(static_cast<unsigned>(windows * (kHkv / heads))), dim3(256), 0, stream, a,
                       heads);
    return hipGetLastError();
}

hipError_t launch_q8_append(const Q8AppendArgs& a, int format, hipStream_t stream) {
    return format == kQ8E4m3 ? launch_append<kQ8E4m3>(a, stream) : launch_append<kQ8Int8>(a, stream);
}

}  // namespace gqa
