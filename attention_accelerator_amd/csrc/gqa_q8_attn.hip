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
//  * Two running references in fp32: m for the scores and M for s + log2(sv).  A weight is formed as
//    w = 2^(s + log2 sv - M) and rounded to fp16 for the products with V's codes: V's scale is
//    inside the weight, and what fp16 loses is relative to the largest w of the column, not to
//    that of a block of a larger scale.  The softmax sum takes 2^(s - m) = w 2^(M - log2 sv - m), one
//    product for the fp32 sum of a lane's eight weights (not the rounded ones: where a block's
//    V scale is small, they hold few bits of s).  O = acc 2^(M - m) / l.
//  * m and M are the maxima as of the last time a key lay more than 2^kSlack above one of them: up to
//    there a weight is at most 2^kSlack, far inside fp16, and nothing has to be rescaled or even
//    compared across lanes.
//  * Keys that a column does not see get w = 0; V rows behind the sequence's end are cleared
//    (they may hold anything, NaN codes too).
#include "gqa_device.h"
#include "gqa_internal.h"
#include "gqa_q8.h"

namespace gqa {

namespace {

constexpr float kLowest = -3.0e38f;        // a reference before any key (finite: no inf - inf)
constexpr float kSlack = 8.0f;             // how far (log2) a key may lie above its reference

// Tokens and first position of sequence b; false where it has no row to compute (lengths that
// break the rules: NaN rows, by the launch that merges).
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

// This lane's part of a query row: dims 16 g .. 16 g + 15 and 64 on, what its B operands hold.
struct Q8Row {
    uint4 lo[2], hi[2];
};

__device__ __forceinline__ Q8Row fetch_q(const uint16_t* row, int g) {
    const uint4* lo = reinterpret_cast<const uint4*>(row + 16 * g);
    const uint4* hi = reinterpret_cast<const uint4*>(row + kPairs + 16 * g);
    return Q8Row{{lo[0], lo[1]}, {hi[0], hi[1]}};
}

// Q operands: B = Q^T of a tile, slice s: lane (g, n) holds column n's dims that lane (g, r) holds of
// a key row: 16 (g + 4 (s / 2)) + 8 (s % 2) + j.  `cs`: (cos, sin) of the column's token in LDS.
// Returns the power of two the row was divided by.
__device__ __forceinline__ float make_q(const Q8AttnArgs& a, const Q8Row& raw, const float2* cs, int g, q8_f16x8 (&op)[4]) {
    float x[16], y[16];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float f[8], e[8];
        unpack8(raw.lo[i], f);
        unpack8(raw.hi[i], e);
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

__device__ __forceinline__ const uint16_t* q_row(const Q8AttnArgs& a, int row, int h, int head) {
    return a.q + static_cast<int64_t>(row) * a.q_token_stride + (kGroup * h + head) * kD;
}

// cos and sin of `tokens` positions from `start` on, by `threads` threads (a token's 64 pairs by
// 64 of them): each thread's first from the angle, the ones after it turned on by the angle of its stride, in
// double (16 turns keep 2^-48 of it; sines of every angle: 2 us more for 64 sequences of 8 tokens).
__device__ __forceinline__ void fill_angles(const Q8AttnArgs& a, int start, int tokens, float2* cs, int tid, int threads) {
    if (!a.rope) return;
    const double f = a.rope_table.inv_freq[tid & 63];
    const int by = threads >> 6;
    double s, c, turn_s = 0.0, turn_c = 1.0;
    rope_sincos(start + (tid >> 6), f, s, c);
    if (tokens > by) rope_sincos(by, f, turn_s, turn_c);
    for (int t = tid >> 6; t < tokens; t += by) {
        cs[t * kPairs + (tid & 63)] = make_float2(static_cast<float>(c), static_cast<float>(s));
        const double u = c * turn_c - s * turn_s;
        s = s * turn_c + c * turn_s;
        c = u;
    }
}

// 16 (or 4) bytes per lane straight into LDS, lane l's at dst + 16 l (4 l): global_load_lds_*.  Inline,
// so that the compiler does not make every later LDS read wait for all copies in flight; the
// waits are explicit (wait_copies).
template <bool kStream>
__device__ __forceinline__ void copy16(const uint8_t* base, uint32_t off, q8_lds* dst) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    if constexpr (kStream)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(at) : "memory");
    else
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(at) : "memory");
}

__device__ __forceinline__ void copy4(const void* src, q8_lds* dst) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "{m0}"(at) : "memory");
}

// Until at most kLeft of this wave's memory operations (copies, and any the compiler issued since)
// are in flight: they end in the order they were issued in.
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

// This lane's reads of a step's planes.  K: row 8 (r / 4) + r % 4 (tile 1: 4 rows on), chunks g and
// g + 4.  V, transposed reads: of each 16 lanes, lane r names 8 bytes of row 8g + r / 2 and gets
// dim r of the 8 rows.
__device__ __forceinline__ uint32_t k_offset(int lane) {
    const int g = lane >> 4, r = lane & 15, row = 8 * (r >> 2) + (r & 3);
    return static_cast<uint32_t>(row * kQ8RowB + 16 * (g ^ k_swizzle(row)));
}

__device__ __forceinline__ uint32_t v_offset(int lane) {
    const int g = lane >> 4, r = lane & 15, row = 8 * g + (r >> 1);
    return static_cast<uint32_t>(row * kQ8RowB + 8 * (r & 1) + 16 * v_swizzle(row));
}

__device__ __forceinline__ q8_i32x2 read_v(const q8_lds* vp, uint32_t voff, int dt) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((GQA_LDS q8_i32x2*)(vp + (voff ^ (16u * dt))));
}

// V of a step that some column does not see whole: rows behind `last` are cleared (they may hold
// anything), and NaN codes, of which 0 * NaN would reach the columns that do not see their key,
// are cleared too, after the elements of the columns that do see them have been marked.  (One-wave workgroups.)
template <int kFmt, int kTiles>
__device__ __forceinline__ void mask_values(q8_lds* vp, int key0, int last, const int (&lim)[kTiles], int lane,
                                            Q8State<kTiles>& st) {
    const int g = lane >> 4;
    for (int row = lane >> 3; row < kQ8Step; row += kWave >> 3)
        if (key0 + row > last) *(GQA_LDS q8_u32x4*)(vp + row * kQ8RowB + 16 * (lane & 7)) = q8_u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    if constexpr (kFmt == kQ8E4m3) {
        uint32_t any = 0;
        for (int row = lane >> 3; row < kQ8Step; row += kWave >> 3) {
            const q8_u32x4 w = *(GQA_LDS q8_u32x4*)(vp + row * kQ8RowB + 16 * (lane & 7));
            any |= nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w);
        }
        if (!__any(any != 0)) return;
        const uint32_t voff = v_offset(lane);
#pragma unroll 1
        for (int dt = 0; dt < 8; ++dt) {
            const q8_i32x2 v = read_v(vp, voff, dt);
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
        for (int row = lane >> 3; row < kQ8Step; row += kWave >> 3) {
            GQA_LDS q8_u32x4* at = (GQA_LDS q8_u32x4*)(vp + row * kQ8RowB + 16 * (lane & 7));
            q8_u32x4 w = *at;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] &= ~(nan_bytes(w[i]) / 0x80u * 0xffu);
            *at = w;
        }
        __syncthreads();
    }
}

// A step's operands as they lie in LDS.  They are read all at once, ahead of their use: left to itself
// the compiler reads each one just before its product and waits for it.
struct Q8KRows {
    q8_u32x4 w[2][2];                      // [tile][chunk g, g + 4]
};

struct Q8VRows {
    q8_i32x2 w[8];                         // [16 dims]
};

__device__ __forceinline__ Q8KRows read_keys(const q8_lds* kp, uint32_t koff) {
    Q8KRows k;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        k.w[t][0] = *(const GQA_LDS q8_u32x4*)(kp + koff + 4 * kQ8RowB * t);
        k.w[t][1] = *(const GQA_LDS q8_u32x4*)(kp + (koff ^ 64u) + 4 * kQ8RowB * t);
    }
    return k;
}

__device__ __forceinline__ Q8VRows read_values(const q8_lds* vp, uint32_t voff) {
    Q8VRows v;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) v.w[dt] = read_v(vp, voff, dt);
    return v;
}

// S^T of 32 keys: s[c][t][i] is the score of key 8g + 4t + i for column n of tile c.
template <int kFmt, int kTiles>
__device__ __forceinline__ void q8_scores(const Q8KRows& k, const q8_f16x8 (&qop)[kTiles][4], f32x4_t (&s)[kTiles][2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const q8_f16x8 k0 = q8_eight<kFmt>(k.w[t][0].x, k.w[t][0].y), k1 = q8_eight<kFmt>(k.w[t][0].z, k.w[t][0].w);
        const q8_f16x8 k2 = q8_eight<kFmt>(k.w[t][1].x, k.w[t][1].y), k3 = q8_eight<kFmt>(k.w[t][1].z, k.w[t][1].w);
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qop[c][0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qop[c][1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k2, qop[c][2], acc, 0, 0, 0);
            s[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k3, qop[c][3], acc, 0, 0, 0);
        }
    }
}

__device__ __forceinline__ float max8(const f32x4_t (&s)[2]) {
    const float a = fmaxf(fmaxf(s[0][0], s[0][1]), s[0][2]), b = fmaxf(fmaxf(s[0][3], s[1][0]), s[1][1]);
    return fmaxf(fmaxf(a, b), fmaxf(s[1][2], s[1][3]));
}

// A step's scores made ready for the weights: keys that a column does not see are -inf, and the
// references move up where one of them has to.  sk, lsv: this lane's block's K scale and log2 of its
// V scale; qs: the columns' powers of two; lim: the last position each column sees; masked: some
// column does not see all 32 keys.
template <int kTiles>
__device__ __forceinline__ void q8_references(f32x4_t (&s)[kTiles][2], float (&f)[kTiles], int key0, bool masked, float sk,
                                              float lsv, const float (&qs)[kTiles], const int (&lim)[kTiles], int lane,
                                              Q8State<kTiles>& st) {
    const int g = lane >> 4;
#pragma unroll
    for (int c = 0; c < kTiles; ++c) f[c] = sk * qs[c];
    if (masked) {
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                s[c][j >> 2][j & 3] = key0 + 8 * g + j <= lim[c] ? s[c][j >> 2][j & 3] * f[c] : -__builtin_inff();
            f[c] = 1.0f;
        }
    }
    float top[kTiles];
    bool over = false;
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
        top[c] = max8(s[c]) * f[c];
        over |= top[c] > st.m[c] + kSlack || top[c] + lsv > st.mv[c] + kSlack;
    }
    if (__any(over)) {
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            const float m = swap32_max(swap16_max(fmaxf(st.m[c], top[c])));
            const float mv = swap32_max(swap16_max(fmaxf(st.mv[c], top[c] + lsv)));
            st.l[c] *= __builtin_amdgcn_exp2f(st.m[c] - m);
            const float down = __builtin_amdgcn_exp2f(st.mv[c] - mv);
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) st.o[c][dt] *= down;
            st.m[c] = m;
            st.mv[c] = mv;
        }
    }
}

// The lane's eight weights of a column as its B operand, and their part of the softmax sum.
template <int kTiles>
__device__ __forceinline__ q8_f16x8 q8_weights(const f32x4_t (&s)[2], float f, float lsv, int c, Q8State<kTiles>& st) {
    // (a V scale 2^100 below the column's others': its weights are 0 in fp16 either way)
    const float base = __builtin_amdgcn_fmed3f(st.mv[c] - lsv, -__builtin_inff(), st.m[c] + 100.0f);
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], f, -base));
    q8_f16x8 p;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const q8_f16x2 two = q8_pack(w[j], w[j + 1]);
        p[j] = two.x;
        p[j + 1] = two.y;
    }
    const float sum = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    st.l[c] = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(base - st.m[c]), st.l[c]);
    return p;
}

// O^T += V^T P^T: A = 16 dims x 32 keys.
template <int kFmt, int kTiles>
__device__ __forceinline__ void q8_values(const Q8VRows& v, const q8_f16x8 (&p)[kTiles], Q8State<kTiles>& st) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
        const q8_f16x8 av = q8_eight<kFmt>(static_cast<uint32_t>(v.w[dt].x), static_cast<uint32_t>(v.w[dt].y));
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
            st.o[c][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, p[c], st.o[c][dt], 0, 0, 0);
    }
}

// Block ids and scales of a (sequence, KV head), 64 blocks (32 steps) at a time: a batch.  They are
// copied into LDS ahead of their use, the ids a batch ahead, the scales when the batch's first step is
// requested.
static __device__ const float kNoScale = __builtin_nanf("");

struct Q8Batch {
    int32_t id[kWave];
    float sk[kWave], sv[kWave];
};
typedef GQA_LDS Q8Batch q8_batch;

// The ids of steps `step` .. `step` + 31 of the sequence with table row `table` and n_blk blocks (past the
// last: its id).
__device__ __forceinline__ void request_ids(q8_batch* bt, const int32_t* table, int step, int n_blk, int lane) {
    copy4(table + min(2 * step + lane, n_blk - 1), (q8_lds*)bt->id);
}

// The scales of a batch whose ids have landed.  An id outside the pool stands for block 0 with a NaN
// scale: the rows that attend to it are NaN.
__device__ __forceinline__ void request_scales(q8_batch* bt, const Q8Pool& pool, int h, int lane) {
    const int32_t id = bt->id[lane];
    const bool ok = id >= 0 && id < pool.n_blocks;
    const int64_t at = id * pool.scale_block_stride + h * pool.scale_head_stride;
    copy4(ok ? pool.k_scale + at : &kNoScale, (q8_lds*)bt->sk);
    copy4(ok ? pool.v_scale + at : &kNoScale, (q8_lds*)bt->sv);
}

__device__ __forceinline__ int64_t batch_block(const q8_batch* bt, const Q8Pool& pool, int step, int which) {
    const int id = __builtin_amdgcn_readfirstlane(bt->id[2 * (step & 31) + which]);
    return id >= 0 && id < pool.n_blocks ? id : 0;
}

// K scale and log2 of the V scale of the lane's block (its keys are 8 (lane / 16) .. of the step).  A
// scale that is negative or NaN makes scores NaN, and with them the rows that attend to it.
__device__ __forceinline__ void batch_scales(const q8_batch* bt, int step, int lane, float& sk, float& lsv) {
    const int at = 2 * (step & 31) + (lane >> 5);
    const float k = bt->sk[at], v = bt->sv[at];
    sk = k >= 0.0f && v >= 0.0f ? k : __builtin_nanf("");
    lsv = __builtin_amdgcn_logf(v >= 0.0f ? v : 0.0f);
}

// Inclusive sum over the wave's lanes (DPP: rows of 16, then the rows' totals handed on).
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, true);      // row_shr:1
    x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, false);     // row_bcast:15 into rows 1, 3
    x += __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, false);     // row_bcast:31 into rows 2, 3
    return x;
}

__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

// The stream: the steps of every sequence of at most kQ8StreamMax rows, laid end to end.  Each KV head
// streams them by itself.  A window is 64 sequences of it, one in each lane.
struct Q8Window {
    int b0;
    Q8Seq seq;                             // this lane's
    int steps;                             // 0: not in the stream
    bool bad;                              // rows to be NaN: its lengths break the rules

    __device__ __forceinline__ void load(const Q8AttnArgs& a, int first, int lane) {
        b0 = first;
        seq = Q8Seq{0, 0, 0};
        steps = 0;
        const bool good = b0 + lane < a.batch && q8_seq(a, b0 + lane, seq);
        if (good && seq.n <= kQ8StreamMax) steps = (seq.start + seq.n + kQ8Step - 1) / kQ8Step;
        bad = !good && seq.n > 0;
    }
};

// How the stream is cut.  Each sequence begins with `lead` positions that hold no step: what starting
// a piece takes (4 us of 1.2 us a step), so that a range which crosses sequences has fewer steps.
// Where sequences are many ranges long there is none: few ranges start one, and ranges that
// divide a length evenly stay aligned with it.
constexpr int kMinRange = 4;               // steps of the smallest range (below, counting and merging costs more)
constexpr int kLead = 3;

struct Q8Cut {
    int64_t total, per;                    // the stream's length, a range's
    int lead;

    __device__ __forceinline__ Q8Cut(int64_t steps, int seqs, int ranges) {
        lead = 4 * static_cast<int64_t>(seqs) > ranges && steps >= 8 * static_cast<int64_t>(ranges) ? kLead : 0;
        total = steps + static_cast<int64_t>(lead) * seqs;
        per = max((total + ranges - 1) / ranges, static_cast<int64_t>(kMinRange));
    }
    // The first and last range that hold steps of a sequence whose step 0 is at position x.
    __device__ __forceinline__ int first_range(int64_t x) const { return static_cast<int>(x / per); }
    __device__ __forceinline__ int last_range(int64_t x, int steps) const { return static_cast<int>((x + steps - 1) / per); }
};

// Partials that another workgroup of the same launch reads go past the L2s, each of which serves one
// XCD: accesses of agent scope (sc1).  (A release fence would write back the whole L2; atomics of 8
// bytes take a cycle of the address unit for each lane: 0.19 us a partial, these 0.02.)
constexpr int kAgentScope = 16;

struct Q8Shared {
    __amdgpu_buffer_rsrc_t rows, ml;

    __device__ __forceinline__ explicit Q8Shared(const Q8AttnArgs& a) {
        const int n = static_cast<int>(2 * a.stream_waves * kGroup);       // partial rows of one-token calls
        rows = __builtin_amdgcn_make_buffer_rsrc(a.part_o, 0, n * kD * 4, 0x00027000);
        ml = __builtin_amdgcn_make_buffer_rsrc(a.part_ml, 0, n * 16, 0x00027000);
    }
    static __device__ __forceinline__ f32x4_t get(__amdgpu_buffer_rsrc_t r, int at) {
        return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kAgentScope));
    }
    static __device__ __forceinline__ void put(__amdgpu_buffer_rsrc_t r, int at, f32x4_t x) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(q8_u32x4, x), r, at, 0, kAgentScope);
    }
};

// NaN rows (of KV head h) for the window's sequences whose lengths break the rules, or that have more than
// max_new rows; none where their offsets do.  By `parts` waves, which deal the rows out; this is wave `part`.
__device__ __forceinline__ void write_nans(const Q8AttnArgs& a, const Q8Window& win, int h, int lane, int part, int parts) {
    for (uint64_t bad = __ballot(win.bad); bad; bad &= bad - 1) {
        const int at = __builtin_ctzll(bad);
        const int row0 = lane_value(win.seq.row0, at), n = lane_value(win.seq.n, at);
        if (row0 < 0 || static_cast<int64_t>(row0) + n > a.n_tokens) continue;
        for (int t = (part + at) % parts; t < n; t += parts) {
            uint16_t* row = a.out + ((static_cast<int64_t>(row0) + t) * kHq + kGroup * h) * kD + 4 * lane;
            *reinterpret_cast<uint2*>(row) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
            *reinterpret_cast<uint2*>(row + kGroup * kD / 2) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
        }
    }
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

// The same rows as partials, row0 + column.  kOne: for this launch's merge.
template <int kTiles, bool kOne>
__device__ __forceinline__ void write_partial(const Q8AttnArgs& a, int64_t row0, int tokens, int lane, Q8State<kTiles>& st) {
    const int g = lane >> 4;
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
        const int col = 16 * c + (lane & 15);
        const float l = cross_row_sum(st.l[c]);
        if ((col >> 2) >= tokens) continue;
        const f32x4_t ml = {st.m[c], st.mv[c], l, 0.0f};
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            f32x4_t o = st.o[c][dt];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = (st.nan[c] >> (4 * dt + i)) & 1 ? __builtin_nanf("") : o[i];
            if constexpr (kOne) Q8Shared::put(Q8Shared(a).rows, static_cast<int>(row0 + col) * kD * 4 + 16 * g + 64 * dt, o);
            else *reinterpret_cast<f32x4_t*>(a.part_o + (row0 + col) * kD + 4 * g + 16 * dt) = o;
        }
        if (g != 0) continue;
        if constexpr (kOne) Q8Shared::put(Q8Shared(a).ml, static_cast<int>(row0 + col) * 16, ml);
        else *reinterpret_cast<f32x4_t*>(a.part_ml + row0 + col) = ml;
    }
}

// out = sum_i O_i 2^(M_i - m) / sum_i l_i 2^(m_i - m) over the n partials of a token's four rows (one KV
// head), by one wave: lane (c, i) has dims 8i .. 8i + 7 of column c.  kBatch partials are in
// flight at once.  row_of(i): partial i's first row.  kOne: of this launch.
template <bool kOne, typename RowOf>
__device__ __forceinline__ void merge_token(const Q8AttnArgs& a, int n, RowOf row_of, uint16_t* out, int lane) {
    constexpr int kBatch = 8;
    const Q8Shared parts(a);
    const int c = lane >> 4, i8 = 8 * (lane & 15);
    float m = kLowest, mv = kLowest, l = 0.0f, o[8] = {};
    for (int i0 = 0; i0 < n; i0 += kBatch) {
        f32x4_t ml[kBatch], x[kBatch][2];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int64_t row = row_of(min(i0 + j, n - 1)) + c;
            if constexpr (kOne) {
                ml[j] = Q8Shared::get(parts.ml, static_cast<int>(row) * 16);
                x[j][0] = Q8Shared::get(parts.rows, (static_cast<int>(row) * kD + i8) * 4);
                x[j][1] = Q8Shared::get(parts.rows, (static_cast<int>(row) * kD + i8) * 4 + 16);
            } else {
                ml[j] = *reinterpret_cast<const f32x4_t*>(a.part_ml + row);
                x[j][0] = *reinterpret_cast<const f32x4_t*>(a.part_o + row * kD + i8);
                x[j][1] = *reinterpret_cast<const f32x4_t*>(a.part_o + row * kD + i8 + 4);
            }
        }
        float top = m, topv = mv;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {         // (a partial past the last is the last again, with no weight)
            top = fmaxf(top, ml[j][0]);
            topv = fmaxf(topv, ml[j][1]);
        }
        const float down = __builtin_amdgcn_exp2f(mv - topv);
        l *= __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] *= down;
        m = top;
        mv = topv;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const float some = i0 + j < n ? 1.0f : 0.0f;
            const float f = some * __builtin_amdgcn_exp2f(ml[j][1] - mv);
            l = __builtin_fmaf(ml[j][2], some * __builtin_amdgcn_exp2f(ml[j][0] - m), l);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[k] = __builtin_fmaf(x[j][0][k], f, o[k]);
                o[4 + k] = __builtin_fmaf(x[j][1][k], f, o[4 + k]);
            }
        }
    }
    const float f = __builtin_amdgcn_exp2f(mv - m) / l;
    *reinterpret_cast<uint4*>(out + c * kD + i8) =
        make_uint4(bf16_pair(o[0] * f, o[1] * f), bf16_pair(o[2] * f, o[3] * f), bf16_pair(o[4] * f, o[5] * f),
                   bf16_pair(o[6] * f, o[7] * f));
}

}  // namespace

// ---------------------------------------------------------------------------------------------
// Stream kernel: sequences of at most kQ8StreamMax new tokens.  Their keys end to end, cut into equal
// ranges, one wave for each range and KV head; the part of a sequence in a range is a piece.  A piece
// that is a whole sequence writes its rows; others leave partials for the merge: slot 2w of the piece
// that enters wave w's range from the one before, 2w + 1 of the one that leaves it.
//
// With one new token for each sequence (kOne) the merge is part of this kernel: the last of a sequence's
// pieces to be written, by a counter in the workspace that it puts back to zero, merges them all.  Of
// more tokens' partials one wave would read up to megabytes: they have a launch of their own.
//
// The eight waves of a range are neighbours, one on each XCD, and read the eight heads' parts of the
// same blocks at about the same time: HBM sees blocks of 16 KB, not 2.
//
// HBM bounds it: 64 sequences of 512..8192 keys, 661 MB, take 112 us, 5.9 TB/s; 8 of 131072, 2.16 GB, 338,
// 6.4 TB/s.  One wave reads a step's eight operands together, before its arithmetic (left in place, each
// waits for LDS: 113 -> 122 us for 8 tokens a sequence).  A single sequence of 4096 keys takes 13 us, its
// ranges 4 steps long: a chain of lengths, ids, scales and keys, and the merge's.
template <int kFmt, int kTiles, bool kOne>
__global__ __launch_bounds__(kWave) __attribute__((amdgpu_waves_per_eu(1)))
void q8_stream_kernel(Q8AttnArgs a) {
    constexpr int kRing = kQ8Ring;
    constexpr int kCopies = 8;                     // memory operations of a step's copies
    constexpr int kBatches = kRing + 1;            // the work's, up to kRing - 1 after it, and the next ids
    __shared__ __align__(4096) uint8_t s_ring[kRing][2][kQ8PlaneB];    // [buffer][K, V]
    __shared__ Q8Batch s_batch[kBatches];
    __shared__ float2 s_cs[kTiles * 4 * kPairs];
    q8_lds* const ring = (q8_lds*)&s_ring[0][0][0];
    q8_batch* const batches = (q8_batch*)&s_batch[0];
    const int lane = threadIdx.x;
    const int wave = blockIdx.x;
    const int h = wave % kHkv;

    // The stream's length, and the sequence at this wave's first position (one window in most batches).
    Q8Window win;
    int64_t all = 0;
    int seqs = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kWave) {
        win.load(a, b0, lane);
        all += static_cast<uint32_t>(lane_value(wave_scan(win.steps), kWave - 1));
        seqs += __popcll(__ballot(win.steps > 0));
        if constexpr (kOne) write_nans(a, win, h, lane, wave / kHkv, a.stream_waves / kHkv);
    }
    // (all lanes store the same: under a branch on the lane the compiler keeps the loop's uniform values in
    // vector registers, 32 more)
    if (!kOne && h == 0) a.cut_seqs[wave / kHkv] = Q8CutSeq{0, 0, 0, 0};
    const Q8Cut cut(all, seqs, a.stream_waves / kHkv);
    int64_t x = wave / kHkv * cut.per;             // next position
    const int64_t x_end = min(x + cut.per, cut.total);
    if (x >= x_end) return;
    int64_t off = 0;                               // position of the window's first sequence
    if (win.b0) win.load(a, 0, lane);
    uint32_t upto = wave_scan(win.steps > 0 ? win.steps + cut.lead : 0);
    uint64_t past;
    while (!(past = __ballot(off + upto > x))) {
        off += static_cast<uint32_t>(lane_value(upto, kWave - 1));
        if (win.b0 + kWave >= a.batch) return;     // (lengths that changed under the call)
        win.load(a, win.b0 + kWave, lane);
        upto = wave_scan(win.steps > 0 ? win.steps + cut.lead : 0);
    }

    // A piece: steps [first, end) of sequence b.  x moves past it.
    struct Piece {
        int b, row0, n, start, first, end, steps;
        int64_t at;                                // position of its sequence's step 0
    };
    auto piece_at = [&](int at, int64_t skip) {    // `skip`: positions of the sequence before x
        Piece p;
        p.at = x - skip + cut.lead;
        p.b = win.b0 + at;
        p.row0 = lane_value(win.seq.row0, at);
        p.n = lane_value(win.seq.n, at);
        p.start = lane_value(win.seq.start, at);
        p.steps = lane_value(win.steps, at);
        p.first = static_cast<int>(max(skip - cut.lead, int64_t{0}));
        const int64_t length = p.steps + cut.lead - skip;
        p.end = static_cast<int>(max(min(x_end - x, length) + skip - cut.lead, int64_t{0}));
        x += length;
        return p;
    };
    // The piece behind p; one without steps where the range ends before it.
    auto piece_after = [&](const Piece& p) {
        uint64_t left = __ballot(win.steps > 0) & ~((2ull << (p.b - win.b0)) - 1);
        while (!left && win.b0 + kWave < a.batch) {
            win.load(a, win.b0 + kWave, lane);
            left = __ballot(win.steps > 0);
        }
        return piece_at(left ? __builtin_ctzll(left) : 0, 0);
    };
    const int at0 = __builtin_ctzll(past);
    Piece cur = piece_at(at0, x - off - static_cast<uint32_t>(lane_value(upto, at0)) + lane_value(win.steps, at0) + cut.lead);
    if (cur.first == cur.end) {                    // the range begins with positions that hold no step
        if (x >= x_end) return;
        cur = piece_after(cur);
        if (cur.first == cur.end) return;
    }

    uint32_t kcopy[4], vcopy[4];                   // this lane's part of a plane's copies, inside its block
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int row = copy_row(q, lane);
        const uint32_t at = static_cast<uint32_t>((row & 15) * a.pool.pos_stride);
        kcopy[q] = at + 16u * ((lane & 7) ^ k_swizzle(row));
        vcopy[q] = at + 16u * ((lane & 7) ^ v_swizzle(row));
    }
    const uint32_t koff = k_offset(lane), voff = v_offset(lane);
    const uint8_t* kh = a.pool.k + h * a.pool.head_stride;
    const uint8_t* vh = a.pool.v + h * a.pool.head_stride;

    // Requests run up to kRing - 1 steps ahead of the work, into the next piece too.  Both sides take the
    // batches in the same order, in the slots of s_batch in turn.
    Piece feed = cur, next = cur;                  // the piece requests are made for; the piece after cur
    bool have_next = x < x_end, feed_next = false; // feed is `next`
    if (have_next) {
        next = piece_after(cur);
        have_next = next.end > 0;
    }
    int feed_step = cur.first, batch_end = cur.first;      // the next step to request; where its batch ends
    int feed_slot = kBatches - 1, feed_buf = 0, ahead = 0;
    bool ids_due = false;                          // the ids of the next batch are not requested: its piece is not known yet
    int since = 0;                                 // steps requested since the last ids were
    auto following = [](int slot) { return slot + 1 == kBatches ? 0 : slot + 1; };
    auto ids = [&](const Piece& p, int n) {
        request_ids(batches + following(feed_slot), a.block_table + static_cast<int64_t>(p.b) * a.max_blocks, 32 * n,
                    (p.start + p.n - 1) / kQ8Block + 1, lane);
        since = 0;
    };
    auto request = [&]() {
        if (feed_step == batch_end) {
            if (feed_step == feed.end) {
                if (!have_next || feed_next) return false;
                feed = next;
                feed_next = true;
                feed_step = 0;
            }
            if (since >= 2) wait_copies<2 * kCopies>();    // the ids have landed
            else if (since == 1) wait_copies<kCopies>();
            else wait_copies<0>();
            feed_slot = following(feed_slot);
            request_scales(batches + feed_slot, a.pool, h, lane);
            const int n = feed_step / 32 + 1;
            batch_end = min(32 * n, feed.end);
            ids_due = false;
            if (32 * n < feed.end) ids(feed, n);
            else if (have_next && !feed_next) ids(next, 0);
            else ids_due = true;
        }
        const q8_batch* bt = batches + feed_slot;
        const int64_t id0 = batch_block(bt, a.pool, feed_step, 0), id1 = batch_block(bt, a.pool, feed_step, 1);
        q8_lds* dst = ring + feed_buf * 2 * kQ8PlaneB;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const uint8_t* base = kv ? vh : kh;
            const uint8_t* b0 = base + id0 * a.pool.block_stride;
            const uint8_t* b1 = base + id1 * a.pool.block_stride;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                copy16<true>(q < 2 ? b0 : b1, (kv ? vcopy : kcopy)[q], dst + kv * kQ8PlaneB + q * 1024);
        }
        feed_buf = feed_buf + 1 == kRing ? 0 : feed_buf + 1;
        ++feed_step;
        ++ahead;
        ++since;
        return true;
    };

    auto wait_steps = [&](int left) {              // until at most `left` steps' copies are in flight
        if (kRing > 3 && left >= 3) wait_copies<3 * kCopies>();
        else if (kRing > 2 && left >= 2) wait_copies<2 * kCopies>();
        else if (left >= 1) wait_copies<kCopies>();
        else wait_copies<0>();
    };

    // The wave's unfinished sequences (kOne): the one its range begins inside of, and the one it ends in.
    struct Part {
        int b, row0, r0, n;                        // the first of the sequence's n pieces is of range r0; n = 0: none
    };
    Part entering{0, 0, 0, 0}, leaving{0, 0, 0, 0};

    ids(cur, cur.first / 32);
    int slot = 0, buf = 0;
    // The piece cur, of at most 4 kNow tokens.  The kernel of four column tiles meets many single tokens
    // (decodes beside prompt chunks) and works on their one tile alone: 87 -> 68 us for 22 decodes and two
    // chunks of 301 tokens.  (Two tiles stay within the time of the reads: 113 us either way for 64
    // sequences of 8 tokens over 512..8192.)
    auto work = [&](auto now) {
        constexpr int kNow = decltype(now)::value;
        Q8State<kNow> st;
        Q8Row raw[kNow];
#pragma unroll
        for (int c = 0; c < kNow; ++c) {
            const int col = 16 * c + (lane & 15);
            raw[c] = fetch_q(q_row(a, cur.row0 + min(col >> 2, cur.n - 1), h, col & 3), lane >> 4);
        }
        while (ahead < kRing - 1 && request()) {}
        fill_angles(a, cur.start, cur.n, s_cs, lane, kWave);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        q8_f16x8 qop[kNow][4];
        float qs[kNow];
        int lim[kNow];
#pragma unroll
        for (int c = 0; c < kNow; ++c) {
            const int tok = min((16 * c + (lane & 15)) >> 2, cur.n - 1);
            qs[c] = make_q(a, raw[c], s_cs + tok * kPairs, lane >> 4, qop[c]);
            lim[c] = cur.start + tok;
        }
        st.clear();
        for (int step = cur.first; step < cur.end; ++step) {
            request();
            wait_steps(ahead - 1);
            const q8_lds* kp = ring + buf * 2 * kQ8PlaneB;
            q8_lds* vp = ring + buf * 2 * kQ8PlaneB + kQ8PlaneB;
            buf = buf + 1 == kRing ? 0 : buf + 1;
            const int key0 = step * kQ8Step;
            const bool masked = key0 + kQ8Step - 1 > cur.start;
            if (masked) mask_values<kFmt, kNow>(vp, key0, cur.start + cur.n - 1, lim, lane, st);
            const Q8KRows k = read_keys(kp, koff);
            float sk, lsv;
            batch_scales(batches + slot, step, lane, sk, lsv);
            const Q8VRows v = read_values(vp, voff);
            __builtin_amdgcn_sched_barrier(0);
            f32x4_t s[kNow][2];
            q8_scores<kFmt, kNow>(k, qop, s);
            float f[kNow];
            q8_references<kNow>(s, f, key0, masked, sk, lsv, qs, lim, lane, st);
            q8_f16x8 p[kNow];
#pragma unroll
            for (int c = 0; c < kNow; ++c) p[c] = q8_weights<kNow>(s[c], f[c], lsv, c, st);
            q8_values<kFmt, kNow>(v, p, st);
            if ((step & 31) == 31 || step + 1 == cur.end) slot = following(slot);
            --ahead;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the buffer's reads are done before it is refilled
        }
        const Q8Seq sq{cur.row0, cur.n, cur.start};
        if (cur.first == 0 && cur.end == cur.steps) {
            write_out<kNow>(a, sq, 0, h, lane, st);
        } else {
            constexpr int kCols = kOne ? kGroup : 16 * kTiles;
            write_partial<kNow, kOne>(a, (2 * static_cast<int64_t>(wave) + (cur.first == 0 ? 1 : 0)) * kCols, cur.n, lane, st);
            if constexpr (kOne) {                  // counted when the wave has no more to request
                const int r0 = cut.first_range(cur.at), n = cut.last_range(cur.at, cur.steps) - r0 + 1;
                (cur.first == 0 ? leaving : entering) = Part{cur.b, cur.row0, r0, n};
            }
        }
    };
    while (true) {
        if (!kOne && cur.first == 0 && cur.end < cur.steps && h == 0)
            a.cut_seqs[wave / kHkv] = Q8CutSeq{cur.row0, cur.n, cur.at + cur.steps - x_end, cut.per};
        if (kTiles == 4 && cur.n <= 4) work(std::integral_constant<int, 1>{});
        else work(std::integral_constant<int, kTiles>{});
        if (!have_next) break;
        cur = next;                                // (which the last request has entered: feed is `cur` now)
        feed_next = false;
        have_next = x < x_end;
        if (have_next) {
            next = piece_after(cur);
            have_next = next.end > 0;
        }
        if (have_next && ids_due) ids(next, 0);
        ids_due = false;
    }
    if constexpr (kOne) {
        if (entering.n == 0 && leaving.n == 0) return;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // the partials are written before they count
        const Part mine = lane == 0 ? entering : leaving;
        uint32_t* counter = a.counters + h * kQ8MaxBatch + mine.b;
        uint32_t done = 0;
        if (lane < 2 && mine.n) done = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
        uint64_t last = __ballot(lane < 2 && mine.n && done == static_cast<uint32_t>(mine.n));
        asm volatile("" ::: "memory");
        if ((last >> lane) & 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (; last; last &= last - 1) {
            const Part part = (last & 1) ? entering : leaving;
            auto row_of = [&](int i) {
                return (2 * (static_cast<int64_t>(part.r0 + i) * kHkv + h) + (i == 0 ? 1 : 0)) * kGroup;
            };
            merge_token<true>(a, part.n, row_of, a.out + (static_cast<int64_t>(part.row0) * kHq + kGroup * h) * kD, lane);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Tile kernel: sequences of more than kQ8StreamMax new tokens, in tiles of 64 tokens (256 columns of one
// KV head) per workgroup of 8 waves, 8 tokens (two column tiles) each.  Two waves share a SIMD: one's
// products run under the other's exponentials.
//
// The workgroup converts K and V to fp16 once for its eight waves, two steps (a stage) at a time:
// each thread takes 16 codes of K and of V, read into registers a stage or two ahead, and writes them
// to the other of two fp16 buffers, with one barrier a stage.  The first wave of a SIMD converts
// at a stage's end and the second at its start: that keeps their products and exponentials apart (303 us
// where both convert at the end: 308).  Where the tiles do not fill the workgroups their keys are cut
// into runs.
//
// 4 sequences with chunks of 512 tokens over 8192 take 306 us: 928 TFLOP/s of products.  A step of 32 keys
// takes a SIMD 2350 clocks: 1024 of products, about 1600 of vector issue (exponentials, sums, conversions), 1024
// of the CU's LDS reads; the two waves overlap them only in part.  (Codes in LDS that every wave converts for
// itself: 348 us; only V as codes: 337; four waves of four column tiles, a SIMD each: 480; the second wave
// half a step behind the first, with three buffers: 357, it spills; higher priority for products: 323.)
constexpr int kTileWaves = 8;
constexpr int kTileCols = kQ8TileTokens * kGroup;
constexpr int kTileRowB = 2 * kD;          // bytes of a row in fp16
constexpr int kTilePlaneB = kQ8Step * kTileRowB;       // K (or V) of a step in fp16
constexpr int kTileMinRun = 4;             // steps of the shortest run (40 tokens over 1000: 24 us, of 8: 28)

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
__device__ __forceinline__ int tile_runs(int tiles, int wgs) { return max(1, wgs / (max(1, min(tiles, wgs)) * kHkv)); }

// Steps of a run of a tile of `steps` steps.
__device__ __forceinline__ int run_steps(int steps, int runs) { return max(kTileMinRun, (steps + runs - 1) / runs); }

__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

typedef short q8_i16x4 __attribute__((ext_vector_type(4)));

// Rows of 256 bytes in 16 chunks of 16.  K: chunk c of row r sits at c ^ k_swizzle(r); V: the 32 bytes
// of 16 dims, number d, at d ^ (r & 7): the rows that one operand read touches together lie in
// different banks.
//
// This lane's reads: K row as in the 8-bit planes, slice s (8 dims: chunk 2 (g + 4 (s / 2)) + s % 2) by
// exclusive or; V, transposed: of each 16 lanes, lane r names 8 bytes of row 8g + r / 4 (and of
// the row 4 on) and gets dim r of the 4 rows.
__device__ __forceinline__ uint32_t k16_offset(int lane) {
    const int g = lane >> 4, r = lane & 15, row = 8 * (r >> 2) + (r & 3);
    return static_cast<uint32_t>(row * kTileRowB + 16 * ((2 * g) ^ k_swizzle(row)));
}

__device__ __forceinline__ uint32_t v16_offset(int lane) {
    const int g = lane >> 4, r = lane & 15, row = 8 * g + (r >> 2);
    return static_cast<uint32_t>(row * kTileRowB + 32 * (row & 7) + 8 * (r & 3));
}

__device__ __forceinline__ q8_f16x8 read_k16(const q8_lds* kp, uint32_t koff, int t, int s) {
    return *(const GQA_LDS q8_f16x8*)(kp + (koff ^ (16u * (s & 1) + 128u * (s >> 1))) + 4 * kTileRowB * t);
}

__device__ __forceinline__ q8_f16x8 read_v16(const q8_lds* vp, uint32_t voff, int dt) {
    const uint32_t at = voff ^ (32u * dt);
    struct {
        q8_i16x4 lo, hi;
    } two = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((GQA_LDS q8_i16x4*)(vp + at)),
             __builtin_amdgcn_ds_read_tr16_b64_v4i16((GQA_LDS q8_i16x4*)(vp + (at ^ 128u) + 4 * kTileRowB))};
    return __builtin_bit_cast(q8_f16x8, two);
}

// As mask_values, of a V plane in fp16 whose rows behind the sequence's end are zero already: NaNs are
// marked for the columns that see them and cleared.
template <int kTiles>
__device__ __forceinline__ void mask_nan16(q8_lds* vp, int key0, const int (&lim)[kTiles], int tid, Q8State<kTiles>& st) {
    const int lane = tid & (kWave - 1), g = lane >> 4;
    bool any = false;
    for (int i = lane; i < kTilePlaneB / 16; i += kWave) {
        const q8_f16x8 x = *(const GQA_LDS q8_f16x8*)(vp + 16 * i);
#pragma unroll
        for (int j = 0; j < 8; ++j) any |= x[j] != x[j];
    }
    if (!__any(any)) return;                       // (the same for every wave: each looked at the whole plane)
    const uint32_t voff = v16_offset(lane);
#pragma unroll 1
    for (int dt = 0; dt < 8; ++dt) {
        const q8_f16x8 x = read_v16(vp, voff, dt);
        q8_f16x8 is;
#pragma unroll
        for (int j = 0; j < 8; ++j) is[j] = x[j] != x[j] ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            q8_f16x8 sees;
#pragma unroll
            for (int j = 0; j < 8; ++j) sees[j] = key0 + 8 * g + j <= lim[c] ? (_Float16)1.0f : (_Float16)0.0f;
            const f32x4_t count = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, sees, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) st.nan[c] |= (count[i] > 0.0f ? 1u : 0u) << (4 * dt + i);
        }
    }
    tile_barrier();
    for (int i = tid; i < kTilePlaneB / 16; i += kTileWaves * kWave) {
        GQA_LDS q8_f16x8* at = (GQA_LDS q8_f16x8*)(vp + 16 * i);
        q8_f16x8 x = *at;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] != x[j] ? (_Float16)0.0f : x[j];
        *at = x;
    }
    tile_barrier();
}

}  // namespace

template <int kFmt>
__global__ __launch_bounds__(kTileWaves * kWave) __attribute__((amdgpu_waves_per_eu(2))) void q8_tile_kernel(Q8AttnArgs a) {
    constexpr int kTiles = 2;
    constexpr int kTokens = 4 * kTiles;            // of a wave
    __shared__ __align__(4096) uint8_t s_stage[2][2][2][kTilePlaneB];          // [buffer][step][K, V]
    __shared__ Q8Batch s_batch[2];
    __shared__ float2 s_cs[kQ8TileTokens * kPairs];
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    q8_lds* const stages = (q8_lds*)&s_stage[0][0][0][0];
    q8_batch* const batches = (q8_batch*)&s_batch[0];
    const int tiles = count_tiles(a, lane);
    const int runs = tile_runs(tiles, a.tile_wgs);
    // This thread's part of a stage: 16 codes of row tid / 8, chunk tid % 8.  (A wave's 8 rows lie in one
    // block, the stage's wv / 2.)
    const int row = tid >> 3, chunk = tid & 7, row32 = row & 31;
    const uint32_t src = static_cast<uint32_t>((row & 15) * a.pool.pos_stride + 16 * chunk);
    const uint32_t kdst = (row >> 5) * 2 * kTilePlaneB + row32 * kTileRowB + 16 * ((2 * chunk) ^ k_swizzle(row32));
    const uint32_t vdst = (row >> 5) * 2 * kTilePlaneB + kTilePlaneB + row32 * kTileRowB + 32 * (chunk ^ (row32 & 7));
    const uint32_t koff = k16_offset(lane), voff = v16_offset(lane);
    const bool late = wv >= kTileWaves / 2;            // the second wave of each SIMD
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
        // Reads the stage of steps first + i and first + i + 1 (a step past the end reads the last block
        // again; it is not used).  Batch n is steps first + 32 n on; wave 0 brings it, its ids a batch
        // ahead, its scales with its first stage.
        uint4 rk, rv;
        auto read = [&](int i) {
            q8_batch* bt = batches + ((i >> 5) & 1);
            if (wv == 0 && (i & 31) == 0) {
                request_scales(bt, a.pool, h, lane);
                request_ids(batches + (~(i >> 5) & 1), table, first + i + 32, n_blk, lane);
            }
            const int64_t at = batch_block(bt, a.pool, i + (wv >> 2), (wv >> 1) & 1) * a.pool.block_stride;
            rk = *reinterpret_cast<const uint4*>(kh + at + src);
            rv = *reinterpret_cast<const uint4*>(vh + at + src);
        };
        // ... and writes it as fp16, V rows behind the last key as zeros.
        auto convert = [&](int i) {
            if ((first + i) * kQ8Step + row > last) rv = make_uint4(0u, 0u, 0u, 0u);
            q8_lds* dst = stages + ((i >> 1) & 1) * 4 * kTilePlaneB;
            *(GQA_LDS q8_f16x8*)(dst + kdst) = q8_eight<kFmt>(rk.x, rk.y);
            *(GQA_LDS q8_f16x8*)(dst + (kdst ^ 16u)) = q8_eight<kFmt>(rk.z, rk.w);
            *(GQA_LDS q8_f16x8*)(dst + vdst) = q8_eight<kFmt>(rv.x, rv.y);
            *(GQA_LDS q8_f16x8*)(dst + vdst + 16) = q8_eight<kFmt>(rv.z, rv.w);
        };
        tile_barrier();                            // (the item before is done with the buffers and the angles)
        if (wv == 0) {
            request_ids(batches, table, first, n_blk, lane);
            wait_copies<0>();
        }
        tile_barrier();
        read(0);
        fill_angles(a, sq.start + tok0, tokens, s_cs, tid, kTileWaves * kWave);
        tile_barrier();
        Q8State<kTiles> st;
        q8_f16x8 qop[kTiles][4];
        float qs[kTiles];
        int lim[kTiles];
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
            const int col = 16 * c + (lane & 15), tok = min(kTokens * wv + (col >> 2), tokens - 1);
            const Q8Row raw = fetch_q(q_row(a, sq.row0 + tok0 + tok, h, col & 3), lane >> 4);
            qs[c] = make_q(a, raw, s_cs + tok * kPairs, lane >> 4, qop[c]);
            lim[c] = sq.start + tok0 + tok;
        }
        st.clear();
        convert(0);
        if (late && first + 2 < end) read(2);
        if (wv == 0) wait_copies<0>();             // the first batch's scales
        tile_barrier();
        for (int step0 = first; step0 < end; step0 += 2) {
            const bool more = step0 + 2 < end;
            if (late) {
                if (more) convert(step0 + 2 - first);
                if (step0 + 4 < end) read(step0 + 4 - first);
            } else if (more) {
                read(step0 + 2 - first);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int step = step0 + e;
                if (step >= end) break;
                q8_lds* kp = stages + ((((step0 - first) >> 1) & 1) * 4 + e * 2) * kTilePlaneB;
                q8_lds* vp = kp + kTilePlaneB;
                const int key0 = step * kQ8Step;
                const bool masked = key0 + kQ8Step - 1 > sq.start + tok0;
                if (kFmt == kQ8E4m3 && masked) mask_nan16<kTiles>(vp, key0, lim, tid, st);
                float sk, lsv;
                batch_scales(batches + (((step - first) >> 5) & 1), step - first, lane, sk, lsv);
                f32x4_t s[kTiles][2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    q8_f16x8 k[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) k[q] = read_k16(kp, koff, t, q);
#pragma unroll
                    for (int c = 0; c < kTiles; ++c) {
                        f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[q], qop[c][q], acc, 0, 0, 0);
                        s[c][t] = acc;
                    }
                }
                float f[kTiles];
                q8_references<kTiles>(s, f, key0, masked, sk, lsv, qs, lim, lane, st);
                q8_f16x8 p[kTiles];
#pragma unroll
                for (int c = 0; c < kTiles; ++c) p[c] = q8_weights<kTiles>(s[c], f[c], lsv, c, st);
                q8_f16x8 v[8];
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) v[dt] = read_v16(vp, voff, dt);
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                    for (int c = 0; c < kTiles; ++c)
                        st.o[c][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[dt], p[c], st.o[c][dt], 0, 0, 0);
            }
            if (more) {
                if (!late) convert(step0 + 2 - first);
                if (wv == 0 && ((step0 + 2 - first) & 31) == 0) wait_copies<0>();      // the batch's scales
                tile_barrier();
            }
        }
        if (wv == 0) wait_copies<0>();             // (ids requested past the end)
        if (per >= steps) {
            write_out<kTiles>(a, sq, tok0 + kTokens * wv, h, lane, st);
        } else {
            const int64_t slot = (static_cast<int64_t>(tile) * kHkv + h) * runs + run;
            write_partial<kTiles, false>(a, a.tile_slot0 + slot * kTileCols + 16 * kTiles * wv, tokens - kTokens * wv, lane, st);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Merge kernel: up to kRangeMergeWaves for each (range, KV head), which share the tokens of the sequence that
// begins in the range and goes on behind it: the first `stream` workgroups.  (The stream kernel names that
// sequence in the workspace.  Found here, by every wave through all lengths, it took 470 us of 1240 for 4096
// sequences of 2 tokens over 512, now 830.)  Then kTileMergeWaves for each (tile, KV head), its tokens in
// turn.  A KV head's waves run on one XCD, the one whose waves wrote its partials (its L2 may still hold
// them).
constexpr int kRangeMergeWaves = 4;          // (1, 2, 8: 122, 116, 114 us for 64 sequences of 8 tokens; 4: 114)
constexpr int kTileMergeWaves = 32;          // (16: 1.2 us more for two chunks of 301 tokens)

__global__ __launch_bounds__(kWave) void q8_merge_kernel(Q8AttnArgs a, int cols, int stream, int waves) {
    const int lane = threadIdx.x;
    const int h = blockIdx.x % kHkv;
    auto out_of = [&](int row) { return a.out + (static_cast<int64_t>(row) * kHq + kGroup * h) * kD; };
    if (static_cast<int>(blockIdx.x) >= stream) {
        const int tiles = count_tiles(a, lane);
        const int runs = tile_runs(tiles, a.tile_wgs);
        const int unit = (blockIdx.x - stream) / kHkv, tile = unit / kTileMergeWaves;
        if (runs == 1 || tile >= tiles) return;
        int b, i;
        find_tile(a, tile, lane, b, i);
        Q8Seq sq;
        q8_seq(a, b, sq);
        const int tokens = min(kQ8TileTokens, sq.n - i * kQ8TileTokens);
        const int steps = (sq.start + i * kQ8TileTokens + tokens - 1) / kQ8Step + 1;
        const int per = run_steps(steps, runs);
        if (per >= steps) return;
        for (int tok = unit % kTileMergeWaves; tok < tokens; tok += kTileMergeWaves) {
            auto row_of = [&](int r) {
                return a.tile_slot0 + ((static_cast<int64_t>(tile) * kHkv + h) * runs + r) * kTileCols + kGroup * tok;
            };
            merge_token<false>(a, (steps + per - 1) / per, row_of, out_of(sq.row0 + i * kQ8TileTokens + tok), lane);
        }
        return;
    }
    const int first = blockIdx.x / kHkv % waves, r0 = blockIdx.x / kHkv / waves;
    const Q8CutSeq seq = a.cut_seqs[r0];
    if (first == 0) {                              // the windows of sequences dealt over the ranges, or the ranges over them
        const int ranges = a.stream_waves / kHkv, windows = (a.batch + kWave - 1) / kWave;
        const int parts = max(1, ranges / windows), part = r0 / windows;
        for (int w = r0 % windows; w < windows && part < parts; w += ranges) {
            Q8Window win;
            win.load(a, w * kWave, lane);
            write_nans(a, win, h, lane, part, parts);
        }
    }
    if (first >= seq.n) return;
    const int pieces = 1 + static_cast<int>((seq.left + seq.per - 1) / seq.per);
    for (int tok = first; tok < seq.n; tok += waves) {
        auto row_of = [&](int i) {
            return (2 * (static_cast<int64_t>(r0 + i) * kHkv + h) + (i == 0 ? 1 : 0)) * static_cast<int64_t>(cols) + kGroup * tok;
        };
        merge_token<false>(a, pieces, row_of, out_of(seq.row0 + tok), lane);
    }
}

template <int kFmt, int kTiles, bool kOne = false>
static void launch_stream(const Q8AttnArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((q8_stream_kernel<kFmt, kTiles, kOne>), dim3(static_cast<unsigned>(a.stream_waves)), dim3(kWave), 0,
                       stream, a);
}

template <int kFmt>
static hipError_t launch_attention(const Q8AttnArgs& a, hipStream_t stream) {
    if (a.max_new == 1) {
        launch_stream<kFmt, 1, true>(a, stream);
        return hipGetLastError();
    }
    const int tiles = q8_stream_tiles(a.max_new);
    if (a.max_new > kQ8StreamMax)
        hipLaunchKernelGGL((q8_tile_kernel<kFmt>), dim3(static_cast<unsigned>(a.tile_wgs)), dim3(kTileWaves * kWave), 0, stream, a);
    if (tiles == 1) launch_stream<kFmt, 1>(a, stream);
    else if (tiles == 2) launch_stream<kFmt, 2>(a, stream);
    else launch_stream<kFmt, 4>(a, stream);
    const int waves = a.max_new < kRangeMergeWaves ? a.max_new : kRangeMergeWaves;
    const int of_stream = a.stream_waves * waves;
    // (runs > 1 only where the tiles and heads are at most half of the workgroups)
    const int of_tiles = a.max_new > kQ8StreamMax ? a.tile_wgs / 2 / kHkv * kHkv * kTileMergeWaves : 0;
    hipLaunchKernelGGL(q8_merge_kernel, dim3(static_cast<unsigned>(of_stream + of_tiles)), dim3(kWave), 0, stream, a, 16 * tiles,
                       of_stream, waves);
    return hipGetLastError();
}

hipError_t launch_q8_attention(const Q8AttnArgs& a, int format, hipStream_t stream) {
    return format == kQ8E4m3 ? launch_attention<kQ8E4m3>(a, stream) : launch_attention<kQ8Int8>(a, stream);
}

}  // namespace gqa
