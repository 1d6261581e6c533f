// gqa_q8_attn.hip -- ragged GQA attention over an 8-bit paged cache on fp16 MFMA.
//
// Row t of sequence b sits at position p_t = seq_len - n + t (n rows) and attends to keys
// p <= p_t:  s_p = scale q . (sk k8_p),  o = sum_p softmax(s)_p (sv v8_p), with sk, sv the scales
// of p's block.
//
// Arithmetic, the same in both kernels, 32 keys (two blocks) at a time:
//  * An 8-bit code is an fp16 number exactly, so K and V enter v_mfma_f32_16x16x32_f16 without a
//    rounding.  Q is rotated (sines and cosines in double, products in fp32), times
//    scale * log2(e), divided by the power of two that brings its row below 1, and rounded to
//    fp16 (2^-12 of an element; the 128 products of a score average it to ~1e-4 of a
//    log2 unit, where the BF16 output rounds at 2e-3).
//  * S^T = K Q^T: A = 16 keys x 32 dims, B = 32 dims x 16 columns.  A column is a (token, head)
//    pair of one KV head: col = 4 token + head.  The rows of the two key tiles are chosen so that
//    lane (g, n) ends with the scores of keys 8g .. 8g+7 of column n: all of one block, so a
//    lane has one sk and one sv, and its eight weights are its B operand of O^T = V^T P^T.
//  * Two running maxima in fp32: m of the scores and M of s + log2(sv).  A weight is formed as
//    w = 2^(s + log2 sv - M) <= 1 and rounded to fp16 for the products with V's codes: V's scale
//    is inside the weight, and what fp16 loses is relative to the largest w of the column, not
//    to that of a block of a larger scale.  The softmax sum takes 2^(s - m) = w 2^(M - log2 sv - m),
//    one product for a lane's eight weights.  O = acc 2^(M - m) / l.
//  * Keys that a column does not see get w = 0; V rows behind the sequence's end are cleared
//    (they may hold anything, NaN codes too).
#include "gqa_device.h"
#include "gqa_internal.h"
#include "gqa_q8.h"

namespace gqa {

namespace {

constexpr float kLowest = -3.0e38f;        // a running max before any key (finite: no inf - inf)

// Tokens and first position of sequence b; false where it has no row to compute (lengths that
// break the rules are the merge kernel's: NaN rows).
struct Q8Seq {
    int row0;      // its first query row
    int n;         // its rows
    int start;     // position of the first
};

__device__ __forceinline__ bool q8_seq(const Q8AttnArgs& a, int b, Q8Seq& s) {
    s.row0 = a.cu ? a.cu[b] : b;
    const int end = a.cu ? a.cu[b + 1] : b + 1;
    const int len = a.seq_len[b];
    s.n = end - s.row0;
    s.start = len - s.n;
    return s.row0 >= 0 && end <= a.n_tokens && s.n > 0 && s.n <= a.max_new && s.start >= 0 &&
           static_cast<int64_t>(len) <= static_cast<int64_t>(a.max_blocks) * kQ8Block;
}

template <int kTiles>
struct Q8State {
    f32x4_t o[kTiles][8];                  // O^T[16 dt + 4 g + i][column n], in units of 2^(M - m)
    float m[kTiles], mv[kTiles], l[kTiles];    // running m and M of the column, this lane's sum
    uint32_t nan[kTiles];                      // bit 4 dt + i: that element's V held a NaN its column sees

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            m[c] = mv[c] = kLowest;
            l[c] = 0.0f;
            nan[c] = 0u;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) o[c][dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
};

// Placement of a row's eight 16-byte chunks in an LDS plane of 32 rows x 128 bytes: chunk c of
// row r sits at position c ^ swizzle(r), chosen so that the 8 rows one operand read touches
// together lie in 8 different positions (K reads rows 8a + b, a and b < 4; V reads 8 rows in turn).
__device__ __forceinline__ int k_swizzle(int r) { return (r & 3) | ((r >> 1) & 4); }
__device__ __forceinline__ int v_swizzle(int r) { return r & 7; }

// Lane l's part of copy q (rows 8q .. 8q+7) of a step's plane.
__device__ __forceinline__ int copy_row(int q, int lane) { return 8 * q + (lane >> 3); }

// Q operands: B = Q^T of tile c, slice s: lane (g, n) holds column n's dims that lane (g, r)
// holds of a key row: 16 (g + 4 (s / 2)) + 8 (s % 2) + j.  `cs`: (cos, sin) of the tile's tokens
// [token][64] in LDS.  Returns the power of two the row was divided by.
__device__ __forceinline__ float load_q(const Q8AttnArgs& a, const uint16_t* row, const float2* cs, int g,
                                        q8_f16x8 (&op)[4]) {
    float x[16], y[16];
    const uint4* lo = reinterpret_cast<const uint4*>(row + 16 * g);
    const uint4* hi = reinterpret_cast<const uint4*>(row + kPairs + 16 * g);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float f[8], e[8];
        unpack8(lo[i], f);
        unpack8(hi[i], e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[8 * i + j] = f[j];
            y[8 * i + j] = e[j];
        }
    }
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        float u = x[j], v = y[j];
        if (a.rope) {
            const float2 t = cs[16 * g + j];
            u = x[j] * t.x - y[j] * t.y;
            v = x[j] * t.y + y[j] * t.x;
        }
        x[j] = u * a.q_scale;
        y[j] = v * a.q_scale;
        top = fmaxf(top, fmaxf(fabsf(x[j]), fabsf(y[j])));
    }
    top = swap32_max(swap16_max(top));
    // 2^e > top (e = exponent + 1), within what an fp32 number and its inverse can be
    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 126, -120), 120);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            op[s][j] = static_cast<_Float16>(x[8 * s + j] * inv);
            op[2 + s][j] = static_cast<_Float16>(y[8 * s + j] * inv);
        }
    return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// cos and sin of `tokens` positions from `start` on, by `threads` threads (a token's 64 pairs by
// 64 of them).
__device__ __forceinline__ void fill_angles(const Q8AttnArgs& a, int start, int tokens, float2* cs, int tid, int threads) {
    if (!a.rope) return;
    const double f = a.rope_table.inv_freq[tid & 63];
    for (int t = tid >> 6; t < tokens; t += threads >> 6) {
        double s, c;
        rope_sincos(start + t, f, s, c);
        cs[t * kPairs + (tid & 63)] = make_float2(static_cast<float>(c), static_cast<float>(s));
    }
}

// 16 bytes per lane straight into LDS (lane l's at dst + 16 l): global_load_lds_dwordx4.  Inline, so
// that the compiler does not make every later LDS read wait for all copies in flight; the
// waits are explicit (wait_copies).
__device__ __forceinline__ void copy16(const uint8_t* base, uint32_t off, const uint8_t* dst, bool stream) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(q8_lds_void*)dst);
    if (stream)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(at) : "memory");
    else
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(at) : "memory");
}

// Until at most kLeft of this wave's memory operations (copies, and any the compiler issued since)
// are in flight.
template <int kLeft>
__device__ __forceinline__ void wait_copies() {
    static_assert(kLeft <= 63, "vmcnt range");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}

// Which bytes of w are NaN codes of e4m3 (0x7f, 0xff): 0x80 in each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
    const uint32_t x = ~w & 0x7f7f7f7fu;           // 0 in a NaN byte
    return ~((x + 0x7f7f7f7fu) | x) & 0x80808080u;
}

// V of a step that some column does not see whole: rows behind `last` are cleared (they may hold
// anything), and NaN codes, of which 0 * NaN would reach the columns that do not see their key,
// are cleared too, after the elements of the columns that do see them have been marked.  Called by
// all `threads` threads of the workgroup.
template <int kFmt, int kTiles>
__device__ __forceinline__ void mask_values(uint8_t* vp, int key0, int last, const int (&lim)[kTiles], int tid, int threads,
                                            Q8State<kTiles>& st) {
    const int lane = tid & (kWave - 1), g = lane >> 4, r = lane & 15;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int row = tid >> 3; row < kQ8Step; row += threads >> 3)
        if (key0 + row > last) *reinterpret_cast<uint4*>(vp + row * kQ8RowB + 16 * (tid & 7)) = zero;
    __syncthreads();
    if constexpr (kFmt == kQ8E4m3) {
        uint32_t any = 0;
        for (int row = lane >> 3; row < kQ8Step; row += kWave >> 3) {
            const uint4 w = *reinterpret_cast<const uint4*>(vp + row * kQ8RowB + 16 * (lane & 7));
            any |= nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w);
        }
        if (!__any(any != 0)) return;              // (the same for every wave: each looked at the whole plane)
        const int vrow = 8 * g + (r >> 1);
#pragma unroll 1
        for (int dt = 0; dt < 8; ++dt) {
            const q8_i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (q8_lds_i32x2*)(vp + vrow * kQ8RowB + 8 * (r & 1) + 16 * (dt ^ v_swizzle(vrow))));
            const uint64_t bits =
                nan_bytes(static_cast<uint32_t>(v.x)) | (static_cast<uint64_t>(nan_bytes(static_cast<uint32_t>(v.y))) << 32);
            q8_f16x8 is;
#pragma unroll
            for (int j = 0; j < 8; ++j) is[j] = (bits >> (8 * j + 7)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
            for (int c = 0; c < kTiles; ++c) {
                q8_f16x8 sees;
#pragma unroll
                for (int j = 0; j < 8; ++j) sees[j] = key0 + 8 * g + j <= lim[c] ? (_Float16)1.0f : (_Float16)0.0f;
                const f32x4_t count =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(is, sees, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) st.nan[c] |= (count[i] > 0.0f ? 1u : 0u) << (4 * dt + i);
            }
        }
        __syncthreads();
        for (int row = tid >> 3; row < kQ8Step; row += threads >> 3) {
            uint4* at = reinterpret_cast<uint4*>(vp + row * kQ8RowB + 16 * (tid & 7));
            uint4 w = *at;
            w.x &= ~(nan_bytes(w.x) / 0x80u * 0xffu);
            w.y &= ~(nan_bytes(w.y) / 0x80u * 0xffu);
            w.z &= ~(nan_bytes(w.z) / 0x80u * 0xffu);
            w.w &= ~(nan_bytes(w.w) / 0x80u * 0xffu);
            *at = w;
        }
        __syncthreads();
    }
}

// One step: 32 keys from position key0 on, in the LDS planes kp and vp.  sk, lsv: this lane's
// block's K scale and log2 of its V scale; qs: the columns' powers of two; lim: the last
// position each column sees; masked: some column does not see all 32 keys.
template <int kFmt, int kTiles>
__device__ __forceinline__ void q8_step(const uint8_t* kp, const uint8_t* vp, int key0, bool masked, float sk, float lsv,
                                        const q8_f16x8 (&qop)[kTiles][4], const float (&qs)[kTiles],
                                        const int (&lim)[kTiles], int lane, Q8State<kTiles>& st) {
    const int g = lane >> 4, r = lane & 15;
    f32x4_t s[kTiles][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int row = 8 * (r >> 2) + (r & 3) + 4 * t;
        const uint8_t* p = kp + row * kQ8RowB;
        const int at = g ^ k_swizzle(row);
        const uint4 w0 = *reinterpret_cast<const uint4*>(p + 16 * at);
        const uint4 w1 = *reinterpret_cast<const uint4*>(p + 16 * (at ^ 4));
        const q8_f16x8 k0 = q8_eight<kFmt>(w0.x, w0.y), k1 = q8_eight<kFmt>(w0.z, w0.w);
        const q8_f16x8 k2 = q8_eight<kFmt>(w1.x, w1.y), k3 = q8_eight<kFmt>(w1.z, w1.w);
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qop[c][0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qop[c][1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k2, qop[c][2], acc, 0, 0, 0);
            s[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k3, qop[c][3], acc, 0, 0, 0);
        }
    }
    // Weights: lane (g, n) has keys key0 + 8g + j.
    q8_f16x8 p[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
        float x[8];
        float f = sk * qs[c];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s[c][j >> 2][j & 3];
        if (masked) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = key0 + 8 * g + j <= lim[c] ? x[j] * f : -__builtin_inff();
            f = 1.0f;
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
        top *= f;
        const float m = swap32_max(swap16_max(fmaxf(st.m[c], top)));
        const float mv = swap32_max(swap16_max(fmaxf(st.mv[c], top + lsv)));
        // (a V scale 2^100 below the column's others': its weights are 0 in fp16 either way)
        const float base = fminf(mv - lsv, m + 100.0f);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], f, -base));
            sum += w;
            p[c][j] = static_cast<_Float16>(w);
        }
        st.l[c] = st.l[c] * __builtin_amdgcn_exp2f(st.m[c] - m) + sum * __builtin_amdgcn_exp2f(base - m);
        if (__any(mv > st.mv[c])) {
            const float down = __builtin_amdgcn_exp2f(st.mv[c] - mv);
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) st.o[c][dt] *= down;
        }
        st.m[c] = m;
        st.mv[c] = mv;
    }
    // O^T += V^T P^T: A = 16 dims x 32 keys by transposed reads of V's rows.
    const int vrow = 8 * g + (r >> 1);
    const uint8_t* vrowp = vp + vrow * kQ8RowB + 8 * (r & 1);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
        const q8_i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32((q8_lds_i32x2*)(vrowp + 16 * (dt ^ v_swizzle(vrow))));
        const q8_f16x8 av = q8_eight<kFmt>(static_cast<uint32_t>(v.x), static_cast<uint32_t>(v.y));
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
            st.o[c][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, p[c], st.o[c][dt], 0, 0, 0);
    }
}

// Block ids and scales of up to 64 blocks (32 steps) of one (sequence, KV head), in LDS.
struct Q8Batch {
    int32_t id[kWave];
    float sk[kWave], sv[kWave];
};

// Fills `bt` for blocks j0 .. j0 + 63 of a sequence with n_blk blocks (past the last: the last).
// An id outside the pool reads block 0 and has a NaN scale, as a block with a scale below zero or
// NaN: the rows that attend to it are NaN.
__device__ __forceinline__ void fill_batch(const Q8AttnArgs& a, const int32_t* table, int h, int j0, int n_blk, int lane,
                                           Q8Batch& bt) {
    const int32_t id = table[min(j0 + lane, n_blk - 1)];
    const bool ok = id >= 0 && id < a.pool.n_blocks;
    const int64_t at = (ok ? id : 0) * a.pool.scale_block_stride + h * a.pool.scale_head_stride;
    const float sk = a.pool.k_scale[at], sv = a.pool.v_scale[at];
    const float nan = __builtin_nanf("");
    bt.id[lane] = ok ? id : 0;
    bt.sk[lane] = ok && sk >= 0.0f && sv >= 0.0f ? sk : nan;               // (NaN scores make the whole row NaN)
    bt.sv[lane] = __builtin_amdgcn_logf(ok && sv >= 0.0f ? sv : 0.0f);     // log2
}

// Where the stream's ranges and segments lie.  The stream is every sequence's steps for KV head 0,
// then 1, ... laid end to end; sequences of more than kQ8StreamMax rows are not in it.
__device__ __forceinline__ int stream_steps(const Q8AttnArgs& a, int b) {
    Q8Seq s;
    if (b >= a.batch || !q8_seq(a, b, s) || s.n > kQ8StreamMax) return 0;
    return (s.start + s.n + kQ8Step - 1) / kQ8Step;
}

// Steps of the whole stream over one KV head.
__device__ int64_t stream_total(const Q8AttnArgs& a, int lane) {
    int64_t sum = 0;
    for (int b = lane; b < a.batch; b += kWave) sum += stream_steps(a, b);
    for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    return sum;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32));
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

constexpr int kMinRange = 2;               // steps of the smallest range

__device__ __forceinline__ int64_t range_steps(int64_t total, int waves) {
    const int64_t per = (total + waves - 1) / waves;
    return per < kMinRange ? kMinRange : per;
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    return f32_to_bf16_rne(lo) | (static_cast<uint32_t>(f32_to_bf16_rne(hi)) << 16);
}

// The finished rows of a piece: out[row][head][dims] = acc 2^(M - m) / l.
template <int kTiles>
__device__ __forceinline__ void write_out(const Q8AttnArgs& a, const Q8Seq& sq, int tok0, int h, int lane, Q8State<kTiles>& st) {
    const int g = lane >> 4;
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
        const int col = 16 * c + (lane & 15), tok = tok0 + (col >> 2);
        const float l = cross_row_sum(st.l[c]);
        const float f = __builtin_amdgcn_exp2f(st.mv[c] - st.m[c]) / l;
        if (tok >= sq.n) continue;
        uint16_t* row = a.out + (static_cast<int64_t>(sq.row0 + tok) * kHq + kGroup * h + (col & 3)) * kD + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            f32x4_t o = st.o[c][dt] * f;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = (st.nan[c] >> (4 * dt + i)) & 1 ? __builtin_nanf("") : o[i];
            *reinterpret_cast<uint2*>(row + 16 * dt) = make_uint2(bf16_pair(o[0], o[1]), bf16_pair(o[2], o[3]));
        }
    }
}

// The same rows as a partial: slot * columns + column.
template <int kTiles>
__device__ __forceinline__ void write_partial(const Q8AttnArgs& a, int64_t row0, int tokens, int lane, Q8State<kTiles>& st) {
    const int g = lane >> 4;
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
        const int col = 16 * c + (lane & 15);
        const float l = cross_row_sum(st.l[c]);
        if ((col >> 2) >= tokens) continue;
        float* row = a.part_o + (row0 + col) * kD + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            f32x4_t o = st.o[c][dt];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = (st.nan[c] >> (4 * dt + i)) & 1 ? __builtin_nanf("") : o[i];
            *reinterpret_cast<f32x4_t*>(row + 16 * dt) = o;
        }
        if (g == 0) a.part_ml[row0 + col] = make_float4(st.m[c], st.mv[c], l, 0.0f);
    }
}

}  // namespace

// ---------------------------------------------------------------------------------------------
// Stream kernel: sequences of at most kQ8StreamMax new tokens.  The keys of every (sequence, KV
// head) end to end, cut into equal ranges, one wave each; the part of a segment in a range is a
// piece.  A piece that is a whole segment writes its rows; others leave partials for the
// merge: slot 2w of the piece that enters range w from the one before, 2w + 1 of the one that
// leaves it.
template <int kFmt, int kTiles>
__global__ __launch_bounds__(kWave) __attribute__((amdgpu_waves_per_eu(kTiles == 4 ? 1 : 2)))
void q8_stream_kernel(Q8AttnArgs a) {
    __shared__ __align__(16) uint8_t s_ring[2][2][kQ8PlaneB];          // [buffer][K, V]
    __shared__ Q8Batch s_batch;
    __shared__ float2 s_cs[kTiles * 4 * kPairs];
    const int lane = threadIdx.x;
    const int64_t per_head = uniform64(stream_total(a, lane));
    const int64_t total = per_head * kHkv;
    const int64_t per = range_steps(total, a.stream_waves);
    const int64_t wave = blockIdx.x;
    int64_t x = wave * per;
    const int64_t x_end = min(x + per, total);
    if (x >= x_end) return;

    // The sequence that holds x: windows of 64 sequences.
    int b = 0, steps = 0;
    int64_t off = 0;                               // stream position of sequence b's first segment
    for (int b0 = 0; b0 < a.batch; b0 += kWave) {
        const int mine = stream_steps(a, b0 + lane);
        int64_t upto = static_cast<int64_t>(mine) * kHkv;
        for (int d = 1; d < kWave; d <<= 1) {
            const int64_t y = __shfl_up(upto, d);
            if (lane >= d) upto += y;
        }
        const uint64_t past = __ballot(off + upto > x);
        if (past) {
            const int at = __builtin_ctzll(past);
            b = b0 + at;
            steps = __builtin_amdgcn_readfirstlane(__shfl(mine, at));
            off += uniform64(__shfl(upto, at)) - static_cast<int64_t>(steps) * kHkv;
            break;
        }
        off += uniform64(__shfl(upto, kWave - 1));
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (steps == 0) return;
    int h = static_cast<int>((x - off) / steps);
    int first = static_cast<int>((x - off) - static_cast<int64_t>(h) * steps);

    uint32_t koff[4], voff[4];                     // this lane's part of a plane's copies, inside its block
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int row = copy_row(q, lane);
        const uint32_t at = static_cast<uint32_t>((row & 15) * a.pool.pos_stride);
        koff[q] = at + 16u * ((lane & 7) ^ k_swizzle(row));
        voff[q] = at + 16u * ((lane & 7) ^ v_swizzle(row));
    }

    Q8State<kTiles> st;
    q8_f16x8 qop[kTiles][4];
    float qs[kTiles];
    int lim[kTiles];
    while (true) {
        Q8Seq sq;
        q8_seq(a, b, sq);
        sq.row0 = __builtin_amdgcn_readfirstlane(sq.row0);
        sq.n = __builtin_amdgcn_readfirstlane(sq.n);
        sq.start = __builtin_amdgcn_readfirstlane(sq.start);
        const int n_steps = static_cast<int>(min(static_cast<int64_t>(steps - first), x_end - x));
        const int end = first + n_steps;
        const int last = sq.start + sq.n - 1;
        const int n_blk = last / kQ8Block + 1;
        const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
        const uint8_t* kh = a.pool.k + h * a.pool.head_stride;
        const uint8_t* vh = a.pool.v + h * a.pool.head_stride;

        auto issue = [&](int step, int buf) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int64_t id = __builtin_amdgcn_readfirstlane(s_batch.id[2 * (step & 31) + (q >> 1)]);
                    copy16((kv ? vh : kh) + id * a.pool.block_stride, (kv ? voff : koff)[q], s_ring[buf][kv] + q * 1024, true);
                }
        };

        fill_batch(a, table, h, 2 * (first & ~31), n_blk, lane, s_batch);
        __syncthreads();
        issue(first, first & 1);
        fill_angles(a, sq.start, sq.n, s_cs, lane, kWave);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            const int col = 16 * c + (lane & 15), tok = min(col >> 2, sq.n - 1);
            qs[c] = load_q(a, a.q + static_cast<int64_t>(sq.row0 + tok) * a.q_token_stride + (kGroup * h + (col & 3)) * kD,
                           s_cs + tok * kPairs, lane >> 4, qop[c]);
            lim[c] = sq.start + tok;
        }
        st.clear();
        for (int step = first; step < end; ++step) {
            const int j = 2 * (step & 31) + (lane >> 5);
            const float sk = s_batch.sk[j], lsv = s_batch.sv[j];
            if (step + 1 < end) {
                if (((step + 1) & 31) == 0) {
                    __syncthreads();
                    fill_batch(a, table, h, 2 * (step + 1), n_blk, lane, s_batch);
                    __syncthreads();
                }
                issue(step + 1, (step + 1) & 1);
                wait_copies<8>();
            } else {
                wait_copies<0>();
            }
            const int key0 = step * kQ8Step;
            const bool masked = key0 + kQ8Step - 1 > sq.start;
            if (masked) mask_values<kFmt, kTiles>(s_ring[step & 1][1], key0, last, lim, lane, kWave, st);
            q8_step<kFmt, kTiles>(s_ring[step & 1][0], s_ring[step & 1][1], key0, masked, sk, lsv, qop, qs, lim, lane, st);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the buffer's reads are done before it is refilled
        }
        if (first == 0 && end == steps)
            write_out<kTiles>(a, sq, 0, h, lane, st);
        else
            write_partial<kTiles>(a, (2 * wave + (first == 0 ? 1 : 0)) * (16 * kTiles), sq.n, lane, st);
        x += n_steps;
        if (x >= x_end) break;
        first = 0;
        if (++h == kHkv) {
            h = 0;
            do {
                ++b;
                steps = __builtin_amdgcn_readfirstlane(stream_steps(a, b));
            } while (steps == 0 && b < a.batch);
            if (steps == 0) break;                 // (lengths that changed under the call)
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// Tile kernel: sequences of more than kQ8StreamMax new tokens, in tiles of 64 tokens (256 columns
// of one KV head) per workgroup of 4 waves, 16 tokens each.  The four waves share the K and V
// steps in LDS.  Where the tiles do not fill the workgroups their keys are cut into runs.
constexpr int kTileWaves = 4;
constexpr int kTileCols = kQ8TileTokens * kGroup;
constexpr int kTileMinRun = 16;            // steps of the shortest run

namespace {

__device__ __forceinline__ int seq_tiles(const Q8AttnArgs& a, int b) {
    Q8Seq s;
    if (b >= a.batch || !q8_seq(a, b, s) || s.n <= kQ8StreamMax) return 0;
    return (s.n + kQ8TileTokens - 1) / kQ8TileTokens;
}

// Tiles of the batch, by every wave for itself.
__device__ int count_tiles(const Q8AttnArgs& a, int lane) {
    int sum = 0;
    for (int b = lane; b < a.batch; b += kWave) sum += seq_tiles(a, b);
    for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    return __builtin_amdgcn_readfirstlane(sum);
}

// The sequence and tile number of tile x of the batch.
__device__ void find_tile(const Q8AttnArgs& a, int x, int lane, int& b, int& i) {
    int off = 0;
    b = i = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kWave) {
        int upto = seq_tiles(a, b0 + lane);
        const int mine = upto;
        for (int d = 1; d < kWave; d <<= 1) {
            const int y = __shfl_up(upto, d);
            if (lane >= d) upto += y;
        }
        const uint64_t past = __ballot(off + upto > x);
        if (past) {
            const int at = __builtin_ctzll(past);
            b = __builtin_amdgcn_readfirstlane(b0 + at);
            i = __builtin_amdgcn_readfirstlane(x - off - __shfl(upto - mine, at));
            return;
        }
        off += __shfl(upto, kWave - 1);
    }
}

// Runs that each tile's keys are cut into: as many as the workgroups can take at once.
__device__ __forceinline__ int tile_runs(int tiles, int wgs) { return max(1, wgs / max(1, tiles * kHkv)); }

// Of a tile of `steps` steps: steps of a run and how many runs hold any.
__device__ __forceinline__ int run_steps(int steps, int runs) { return max(kTileMinRun, (steps + runs - 1) / runs); }

}  // namespace

template <int kFmt>
__global__ __launch_bounds__(kTileWaves * kWave) void q8_tile_kernel(Q8AttnArgs a) {
    __shared__ __align__(16) uint8_t s_ring[2][2][kQ8PlaneB];
    __shared__ Q8Batch s_batch;
    __shared__ float2 s_cs[kQ8TileTokens * kPairs];
    constexpr int kTiles = 4;
    const int lane = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = count_tiles(a, lane);
    const int runs = tile_runs(tiles, a.tile_wgs);
    uint32_t koff, voff;
    {
        const int row = copy_row(wv, lane);
        const uint32_t at = static_cast<uint32_t>((row & 15) * a.pool.pos_stride);
        koff = at + 16u * ((lane & 7) ^ k_swizzle(row));
        voff = at + 16u * ((lane & 7) ^ v_swizzle(row));
    }
    const int64_t items = static_cast<int64_t>(tiles) * kHkv * runs;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int h = static_cast<int>(item % kHkv);
        const int run = static_cast<int>(item / kHkv % runs);
        const int tile = tiles - 1 - static_cast<int>(item / kHkv / runs);
        int b, i;
        find_tile(a, tile, lane, b, i);
        Q8Seq sq;
        q8_seq(a, b, sq);
        sq.row0 = __builtin_amdgcn_readfirstlane(sq.row0);
        sq.n = __builtin_amdgcn_readfirstlane(sq.n);
        sq.start = __builtin_amdgcn_readfirstlane(sq.start);
        const int tok0 = i * kQ8TileTokens;
        const int tokens = min(kQ8TileTokens, sq.n - tok0);
        const int last = sq.start + tok0 + tokens - 1;         // the last key of the tile
        const int steps = last / kQ8Step + 1;
        const int per = run_steps(steps, runs);
        const int first = run * per, end = min(first + per, steps);
        if (first >= end) continue;
        const int n_blk = last / kQ8Block + 1;
        const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
        const uint8_t* kh = a.pool.k + h * a.pool.head_stride;
        const uint8_t* vh = a.pool.v + h * a.pool.head_stride;
        auto issue = [&](int step, int buf) {
            const int64_t id = __builtin_amdgcn_readfirstlane(s_batch.id[2 * (step & 31) + (wv >> 1)]);
            copy16(kh + id * a.pool.block_stride, koff, s_ring[buf][0] + wv * 1024, false);
            copy16(vh + id * a.pool.block_stride, voff, s_ring[buf][1] + wv * 1024, false);
        };
        __syncthreads();
        if (wv == 0) fill_batch(a, table, h, 2 * (first & ~31), n_blk, lane, s_batch);
        fill_angles(a, sq.start + tok0, tokens, s_cs, threadIdx.x, kTileWaves * kWave);
        __syncthreads();
        issue(first, first & 1);
        Q8State<kTiles> st;
        q8_f16x8 qop[kTiles][4];
        float qs[kTiles];
        int lim[kTiles];
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            const int col = 16 * c + (lane & 15), tok = min(16 * wv + (col >> 2), tokens - 1);
            qs[c] = load_q(a, a.q + static_cast<int64_t>(sq.row0 + tok0 + tok) * a.q_token_stride + (kGroup * h + (col & 3)) * kD,
                           s_cs + tok * kPairs, lane >> 4, qop[c]);
            lim[c] = sq.start + tok0 + tok;
        }
        st.clear();
        for (int step = first; step < end; ++step) {
            const int j = 2 * (step & 31) + (lane >> 5);
            const float sk = s_batch.sk[j], lsv = s_batch.sv[j];
            wait_copies<0>();
            __syncthreads();                       // the step has landed, and the other buffer is free
            if (step + 1 < end) {
                if (((step + 1) & 31) == 0) {
                    if (wv == 0) fill_batch(a, table, h, 2 * (step + 1), n_blk, lane, s_batch);
                    __syncthreads();
                }
                issue(step + 1, (step + 1) & 1);
            }
            const int key0 = step * kQ8Step;
            const bool masked = key0 + kQ8Step - 1 > sq.start + tok0;
            if (masked) mask_values<kFmt, kTiles>(s_ring[step & 1][1], key0, last, lim, threadIdx.x, kTileWaves * kWave, st);
            q8_step<kFmt, kTiles>(s_ring[step & 1][0], s_ring[step & 1][1], key0, masked, sk, lsv, qop, qs, lim, lane, st);
        }
        if (per >= steps) {
            write_out<kTiles>(a, sq, tok0 + 16 * wv, h, lane, st);
        } else {
            const int64_t slot = (static_cast<int64_t>(tile) * kHkv + h) * runs + run;
            write_partial<kTiles>(a, a.tile_slot0 + slot * kTileCols + 64 * wv, tokens - 16 * wv, lane, st);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Merge: out = sum_i O_i 2^(M_i - m) / sum_i l_i 2^(m_i - m) over the partials of a row, and NaN
// rows for sequences whose lengths break the rules.
namespace {

// One row by one wave: lane has dims 2 lane, 2 lane + 1.  Partials at row0 + i * stride.
__device__ __forceinline__ void merge_row(const Q8AttnArgs& a, int64_t row0, int64_t first, int64_t stride, int n, uint16_t* out,
                                          int lane) {
    float m = kLowest, mv = kLowest;
    for (int i = lane; i < n; i += kWave) {
        const float4 p = a.part_ml[i == 0 ? first : row0 + (i - 1) * stride];
        m = fmaxf(m, p.x);
        mv = fmaxf(mv, p.y);
    }
    m = wave_max(m);
    mv = wave_max(mv);
    float l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
        const int64_t r = i == 0 ? first : row0 + (i - 1) * stride;
        const float4 p = a.part_ml[r];
        const float2 o = *reinterpret_cast<const float2*>(a.part_o + r * kD + 2 * lane);
        const float f = __builtin_amdgcn_exp2f(p.y - mv);
        l += p.z * __builtin_amdgcn_exp2f(p.x - m);
        x += o.x * f;
        y += o.y * f;
    }
    const float f = __builtin_amdgcn_exp2f(mv - m) / l;
    *reinterpret_cast<uint32_t*>(out + 2 * lane) = bf16_pair(x * f, y * f);
}

}  // namespace

// Grid: (sequence, KV head), groups of 4 columns (one token's).  A wave takes one column.
__global__ __launch_bounds__(kGroup * kWave) void q8_stream_merge_kernel(Q8AttnArgs a, int cols) {
    const int lane = threadIdx.x & (kWave - 1), head = threadIdx.x >> 6;
    const int b = blockIdx.x / kHkv, h = blockIdx.x % kHkv;
    Q8Seq sq;
    if (!q8_seq(a, b, sq)) {
        // Rows of a sequence whose lengths break the rules (or that has more than max_new): NaN.
        if (sq.row0 < 0 || sq.n <= 0 || static_cast<int64_t>(sq.row0) + sq.n > a.n_tokens) return;
        for (int t = blockIdx.y; t < sq.n; t += gridDim.y)
            reinterpret_cast<uint32_t*>(a.out)[((static_cast<int64_t>(sq.row0) + t) * kHq + kGroup * h + head) * (kD / 2) + lane] =
                0x7fc07fc0u;
        return;
    }
    const int tok = blockIdx.y;
    if (sq.n > kQ8StreamMax || tok >= sq.n) return;
    // The segment's place in the stream.
    int64_t off = 0, all = 0;
    for (int i = lane; i < a.batch; i += kWave) {
        const int s = stream_steps(a, i);
        all += s;
        off += i < b ? s : 0;
    }
    for (int d = 1; d < kWave; d <<= 1) {
        all += __shfl_xor(all, d);
        off += __shfl_xor(off, d);
    }
    const int steps = stream_steps(a, b);
    const int64_t per = range_steps(uniform64(all) * kHkv, a.stream_waves);
    const int64_t x = uniform64(off) * kHkv + static_cast<int64_t>(h) * steps;
    const int64_t w0 = x / per, w1 = (x + steps - 1) / per;
    if (w0 == w1) return;                          // one piece: written already
    const int col = kGroup * tok + head;
    merge_row(a, 2 * (w0 + 1) * cols + col, (2 * w0 + 1) * cols + col, 2 * cols, static_cast<int>(w1 - w0 + 1),
              a.out + (static_cast<int64_t>(sq.row0 + tok) * kHq + kGroup * h + head) * kD, lane);
}

// Grid: workgroups of the tile kernel, tokens of a tile.
__global__ __launch_bounds__(kGroup * kWave) void q8_tile_merge_kernel(Q8AttnArgs a) {
    const int lane = threadIdx.x & (kWave - 1), head = threadIdx.x >> 6;
    const int tiles = count_tiles(a, lane);
    const int runs = tile_runs(tiles, a.tile_wgs);
    const int at = blockIdx.x;
    if (runs == 1 || at >= tiles * kHkv) return;
    const int tile = at / kHkv, h = at % kHkv, tok = blockIdx.y;
    int b, i;
    find_tile(a, tile, lane, b, i);
    Q8Seq sq;
    q8_seq(a, b, sq);
    const int t = i * kQ8TileTokens + tok;
    if (t >= sq.n) return;
    const int tokens = min(kQ8TileTokens, sq.n - i * kQ8TileTokens);
    const int steps = (sq.start + i * kQ8TileTokens + tokens - 1) / kQ8Step + 1;
    const int per = run_steps(steps, runs);
    if (per >= steps) return;
    const int64_t row = a.tile_slot0 + static_cast<int64_t>(at) * runs * kTileCols + kGroup * tok + head;
    merge_row(a, row + kTileCols, row, kTileCols, (steps + per - 1) / per,
              a.out + (static_cast<int64_t>(sq.row0 + t) * kHq + kGroup * h + head) * kD, lane);
}

template <int kFmt, int kTiles>
static void launch_stream(const Q8AttnArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((q8_stream_kernel<kFmt, kTiles>), dim3(static_cast<unsigned>(a.stream_waves)), dim3(kWave), 0, stream, a);
}

template <int kFmt>
static hipError_t launch_attention(const Q8AttnArgs& a, hipStream_t stream) {
    const int tiles = q8_stream_tiles(a.max_new);
    if (a.max_new > kQ8StreamMax)
        hipLaunchKernelGGL((q8_tile_kernel<kFmt>), dim3(static_cast<unsigned>(a.tile_wgs)), dim3(kTileWaves * kWave), 0, stream, a);
    if (tiles == 1) launch_stream<kFmt, 1>(a, stream);
    else if (tiles == 2) launch_stream<kFmt, 2>(a, stream);
    else launch_stream<kFmt, 4>(a, stream);
    const int toks = a.max_new < kQ8StreamMax ? a.max_new : kQ8StreamMax;
    hipLaunchKernelGGL(q8_stream_merge_kernel, dim3(static_cast<unsigned>(a.batch) * kHkv, static_cast<unsigned>(toks)),
                       dim3(kGroup * kWave), 0, stream, a, 16 * tiles);
    if (a.max_new > kQ8StreamMax)
        hipLaunchKernelGGL(q8_tile_merge_kernel, dim3(static_cast<unsigned>(a.tile_wgs), kQ8TileTokens),
                           dim3(kGroup * kWave), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_q8_attention(const Q8AttnArgs& a, int format, hipStream_t stream) {
    return format == kQ8E4m3 ? launch_attention<kQ8E4m3>(a, stream) : launch_attention<kQ8Int8>(a, stream);
}

}  // namespace gqa
