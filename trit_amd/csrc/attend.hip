// Attention of a few or many query rows to int8 blocks (a paged cache's full
// ones) and f16 blocks (its open ones, or an encoder's states).
#include <climits>

#include "attend.h"
#include "device.h"

namespace trit {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr int WAVES = 4;
// The largest fixed-point value of three int8 digits, and the factor that
// keeps the low part of an f16 pair clear of subnormal f16.
constexpr float FIXED = 8323072.0f;  // 127 * 65536
constexpr float PAIR = 1024.0f;

// The larger of a value and the one 32 (16) lanes away: a swap of two copies
// leaves a lane its own value in one and the other's in the other.
__device__ __forceinline__ float other_half_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_row_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// The largest over a column's four lanes (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float column_max(float v) { return other_half_max(other_row_max(v)); }
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// The three digits of 4 fixed-point values (|x| <= FIXED), each digit's 4
// bytes in a word: x + 0x808080 carries what a signed digit takes from the
// next one, and flipping the top bits makes the bytes signed.
__device__ __forceinline__ void digits4(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, int& d0, int& d1, int& d2) {
    const uint32_t t0 = (x0 + 0x808080u) ^ 0x808080u, t1 = (x1 + 0x808080u) ^ 0x808080u;
    const uint32_t t2 = (x2 + 0x808080u) ^ 0x808080u, t3 = (x3 + 0x808080u) ^ 0x808080u;
    const uint32_t a = __builtin_amdgcn_perm(t1, t0, 0x05010400u), b = __builtin_amdgcn_perm(t3, t2, 0x05010400u);
    d0 = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
    d1 = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
    const uint32_t c = __builtin_amdgcn_perm(t1, t0, 0x0c0c0602u), d = __builtin_amdgcn_perm(t3, t2, 0x0c0c0602u);
    d2 = (int)__builtin_amdgcn_perm(d, c, 0x05040100u);
}

// A wave's running softmax of 16 columns (query rows of the heads that share
// a key head): lane l holds column l % 16, and of the output the dims
// 16 n + 4 (l / 16) + r.
template <int HDP>
struct Running {
    float m = -INFINITY;  // the largest score so far, in powers of two (the same in a column's lanes)
    float l = 0.0f;       // this lane's part of the sum of 2^(score - m)
    v4f acc[HDP / 16];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < HDP / 16; ++n) acc[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// Scores u * f (f >= 0 or NaN) of a block to probabilities of that block
// alone, p = 2^(u f - max) <= 1, in place; then the running maximum takes the
// block's. `before` scales what was summed, `now` the block's products: a
// block's probabilities are fixed-point values or f16 pairs relative to its
// own maximum, so that a long tail of small ones next to one large one far
// away keeps its digits. seen: the columns' keys from this block on; values
// from there on do not count, whatever they hold.
// Returns whether the column sees any of the block.
template <bool MASK>
__device__ __forceinline__ bool block_softmax(float (&u)[16], float f, int seen, float& m, float& l, float& before,
                                              float& now) {
    const int lq = (threadIdx.x % WAVE) / 16;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (MASK && 16 * (i / 4) + 4 * lq + i % 4 >= seen) u[i] = -INFINITY;
        top = __builtin_fmaxf(top, u[i]);
    }
    top = column_max(top);
    const bool any = !MASK || top > -INFINITY;
    const float mb = any ? top * f : -INFINITY;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        // The difference first: never above 0, whatever the scores' size.
        const float p = __builtin_amdgcn_exp2f((u[i] - top) * f);
        u[i] = MASK && 16 * (i / 4) + 4 * lq + i % 4 >= seen ? 0.0f : p;
        sum += u[i];
    }
    const float mn = __builtin_fmaxf(m, mb);
    before = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    now = any ? __builtin_amdgcn_exp2f(mb - mn) : 0.0f;
    m = mn;
    l = __builtin_fmaf(now, sum, l * before);
    return any;
}

// The columns' queries as fixed point: x = round(q * FIXED / max|q|), three
// digits, and the step max|q| / FIXED (times scale and log2 e).
template <int HDP>
struct Digits {
    v4i d[3][HDP / 64];
    float step;
};

// 16 or 8 consecutive values of a query, 0 past head_dim or for no query.
template <int N>
__device__ __forceinline__ void load_query(const float* q, int e, int hd, float scale, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = q && e + i < hd ? q[e + i] * scale : 0.0f;
}

template <int HDP>
__device__ __forceinline__ void query_digits(const float* q, int hd, float scale, Digits<HDP>& out) {
    const int lq = (threadIdx.x % WAVE) / 16;
    float v[HDP / 64][16], top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int ks = 0; ks < HDP / 64; ++ks) {
        load_query(q, 64 * ks + 16 * lq, hd, scale, v[ks]);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            top = __builtin_fmaxf(top, __builtin_fabsf(v[ks][i]));
            bad |= v[ks][i] != v[ks][i];
        }
    }
    // A query that holds a NaN has NaN scores (a maximum passes over it).
    top = column_max(bad ? INFINITY : top);
    // Queries below 1e-30 have scores that differ by nothing; an infinite
    // one has no digits and NaN scores.
    const float inv = FIXED / __builtin_fmaxf(top, 1e-30f);
    out.step = top < INFINITY ? __builtin_fmaxf(top, 1e-30f) * (1.0f / FIXED) * LOG2E : NAN;
#pragma unroll
    for (int ks = 0; ks < HDP / 64; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float s = __builtin_rintf(v[ks][4 * i + r] * inv);
                x[r] = (uint32_t)(int)__builtin_fminf(__builtin_fmaxf(s, -FIXED), FIXED);
            }
            int d0, d1, d2;
            digits4(x[0], x[1], x[2], x[3], d0, d1, d2);
            out.d[0][ks][i] = d0;
            out.d[1][ks][i] = d1;
            out.d[2][ks][i] = d2;
        }
}

// The columns' queries as pairs of f16 values hi + lo, scaled to a largest
// magnitude of PAIR; step as above.
template <int HDP>
struct Pairs {
    v8h hi[HDP / 32], lo[HDP / 32];
    float step;
};
template <int HDP>
__device__ __forceinline__ void query_pairs(const float* q, int hd, float scale, Pairs<HDP>& out) {
    const int lq = (threadIdx.x % WAVE) / 16;
    float v[HDP / 32][8], top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int ks = 0; ks < HDP / 32; ++ks) {
        load_query(q, 32 * ks + 8 * lq, hd, scale, v[ks]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top = __builtin_fmaxf(top, __builtin_fabsf(v[ks][i]));
            bad |= v[ks][i] != v[ks][i];
        }
    }
    top = column_max(bad ? INFINITY : top);
    const float inv = PAIR / __builtin_fmaxf(top, 1e-30f);
    out.step = top < INFINITY ? __builtin_fmaxf(top, 1e-30f) * (1.0f / PAIR) * LOG2E : NAN;
#pragma unroll
    for (int ks = 0; ks < HDP / 32; ++ks)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = top < INFINITY ? v[ks][i] * inv : 0.0f;
            const _Float16 hi = (_Float16)x;
            out.hi[ks][i] = hi;
            out.lo[ks][i] = (_Float16)(x - (float)hi);
        }
}

// One full block of int8 codes. Both products run in integers: the query and
// the probabilities are three int8 digits each, so their products with the
// codes are exact, and what is rounded is one fixed-point step of 24 bits.
template <int HDP, bool MASK>
__device__ __forceinline__ void codes_block(const uint8_t* block, float2 sc, const Digits<HDP>& qd, int seen,
                                            Running<HDP>& run) {
    constexpr int KS = HDP / 64, NT = HDP / 16;
    const int lane = threadIdx.x % WAVE;
    const uint8_t* at = block + lane * 16;
    v4i kf[4 * KS], vf[NT];
#pragma unroll
    for (int i = 0; i < 4 * KS; ++i) kf[i] = *(const TRIT_GLOBAL v4i*)(at + i * 1024);
#pragma unroll
    for (int i = 0; i < NT; ++i) vf[i] = *(const TRIT_GLOBAL v4i*)(at + BLOCK_TOKENS * HDP + i * 1024);
    float u[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        v4i c[3];
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            c[j] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                c[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t * KS + ks], qd.d[j][ks], c[j], 0, 0, 0);
        }
        // |c| <= 128 * 127 * 128: c1 * 256 + c0 stays within 32 bits.
#pragma unroll
        for (int r = 0; r < 4; ++r)
            u[4 * t + r] = __builtin_fmaf((float)c[2][r], 65536.0f, (float)((c[1][r] << 8) + c[0][r]));
    }
    float before, now;
    const bool any = block_softmax<MASK>(u, qd.step * sc.x, seen, run.m, run.l, before, now);
    v4i pd[3];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        uint32_t x[4];
        // round(p * FIXED) in the low bits of a float of exponent 2^23.
#pragma unroll
        for (int r = 0; r < 4; ++r)
            x[r] = __builtin_bit_cast(uint32_t, __builtin_fmaf(u[4 * t + r], FIXED, 8388608.0f));
        int d0, d1, d2;
        digits4(x[0], x[1], x[2], x[3], d0, d1, d2);
        pd[0][t] = d0;
        pd[1][t] = d1;
        pd[2][t] = d2;
    }
    // A column that sees nothing of the block takes nothing of it, also where its scale is NaN.
    const float w = any ? now * sc.y * (1.0f / FIXED) : 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        v4i c[3];
#pragma unroll
        for (int j = 0; j < 3; ++j)
            c[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[n], pd[j], v4i{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float o = __builtin_fmaf((float)c[2][r], 65536.0f, (float)((c[1][r] << 8) + c[0][r]));
            run.acc[n][r] = __builtin_fmaf(o, w, run.acc[n][r] * before);
        }
    }
}

__device__ __forceinline__ bool any_nan(v8h x) {
    const v4i w = __builtin_bit_cast(v4i, x);
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) hit |= (((uint32_t)w[i] & 0x7fff7fffu) + 0x03ff03ffu) & 0x80008000u;
    return hit != 0;
}

// One f16 block of `tokens` valid ones. CHECK: its values behind the last
// token are left from other sequences, and a NaN among the valid ones counts
// for the columns that see its token and no others.
template <int HDP, bool CHECK>
__device__ __forceinline__ void f16_block(const _Float16* block, int tokens, const Pairs<HDP>& qp, int seen,
                                          Running<HDP>& run) {
    constexpr int KS = HDP / 32, NT = HDP / 16;
    const int lane = threadIdx.x % WAVE, lq = lane / 16;
    const _Float16* at = block + lane * 8;
    v8h kf[4 * KS], vf[NT * 2];
#pragma unroll
    for (int i = 0; i < 4 * KS; ++i) kf[i] = *(const TRIT_GLOBAL v8h*)(at + i * 512);
#pragma unroll
    for (int i = 0; i < NT * 2; ++i) vf[i] = *(const TRIT_GLOBAL v8h*)(at + BLOCK_TOKENS * HDP + i * 512);
    float u[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        v4f c = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t * KS + ks], qp.lo[ks], c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t * KS + ks], qp.hi[ks], c, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) u[4 * t + r] = c[r];
    }
    float before, now;
    const int limit = seen < tokens ? seen : tokens;
    block_softmax<true>(u, qp.step, limit, run.m, run.l, before, now);
    v8h ph[2], pl[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float p = u[i] * PAIR;
        const _Float16 hi = (_Float16)p;
        ph[i / 8][i % 8] = hi;
        pl[i / 8][i % 8] = (_Float16)(p - (float)hi);
    }
    const float w = now * (1.0f / PAIR);
    bool nans = false;
    if (CHECK) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool valid = 32 * s + 16 * (i / 4) + 4 * lq + i % 4 < tokens;
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    if (!valid) vf[2 * n + s][i] = (_Float16)0.0f;
            }
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) nans |= any_nan(vf[i]);
        nans = __ballot(nans) != 0;
    }
    // Which of the lane's tokens its column sees, as f16 ones.
    v8h sees[2];
    if (CHECK && nans) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sees[i / 8][i % 8] = (_Float16)(16 * (i / 4) + 4 * lq + i % 4 < limit ? 1.0f : 0.0f);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        v4f c = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (CHECK && nans) {
            v4f count = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                v8h is;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool nan = vf[2 * n + s][i] != vf[2 * n + s][i];
                    is[i] = (_Float16)(nan ? 1.0f : 0.0f);
                    if (nan) vf[2 * n + s][i] = (_Float16)0.0f;
                }
                count = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, sees[s], count, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (count[r] > 0.0f) c[r] = NAN;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[2 * n + s], pl[s], c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[2 * n + s], ph[s], c, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) run.acc[n][r] = __builtin_fmaf(c[r], w, run.acc[n][r] * before);
    }
}

__global__ void clear_kernel(int* p, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) p[i] = 0;
}

// Words that other workgroups of the launch read: to and from memory past the
// caches that a reader on another XCD does not share.
__device__ __forceinline__ void put(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get(const float* p) {
    const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Block (item): sequence, key head g, a tile of 16 columns (query row r, head
// g * group + c of it: column r * group + c) and a chunk of its key blocks.
// The four waves take the chunk's blocks in turn and join their sums in shared
// memory. Of the workgroups of a tile's chunks the last to end joins theirs,
// in the chunks' order.
template <int HDP, bool PAGED>
__global__ __launch_bounds__(WAVES * WAVE) void attend_kernel(AttendArgs a) {
    constexpr int NT = HDP / 16;
    __shared__ float top[WAVES][16], sum[WAVES][16];
    __shared__ float part[WAVES][16][HDP];
    __shared__ bool arrived;
    const int t = threadIdx.x, w = t / WAVE, lane = t % WAVE, col = lane % 16, lq = lane / 16;
    // The last sequence whose items start at or before this one.
    int si = 0;
#pragma unroll
    for (int i = 0; i < CALL_SEQS; i += WAVE)
        si += __popcll(__ballot(i + lane < a.n && a.s[i + lane].start <= (int)blockIdx.x));
    const AttendSeq seq = a.s[si - 1];
    const int item = (int)blockIdx.x - seq.start;
    const int g = item % a.kv_heads, chunk = item / a.kv_heads % seq.chunks, tile = item / a.kv_heads / seq.chunks;
    const int columns = seq.rows * a.group;
    const int c = tile * 16 + col, row = c / a.group;
    const int head = g * a.group + c % a.group;
    const float* q = c < columns ? a.q + (size_t)(seq.first + row) * a.qs + (size_t)head * a.hd : nullptr;
    // Keys the column sees; the tile's most and least.
    const int ahead = PAGED ? seq.len - seq.rows + 1 : seq.len;
    const int last = (tile * 16 + 15 < columns ? tile * 16 + 15 : columns - 1) / a.group;
    const int most = PAGED ? ahead + last : ahead, least = PAGED ? ahead + tile * 16 / a.group : ahead;
    const int seen = c < columns ? (PAGED ? ahead + row : ahead) : 0;
    const int b0 = chunk * a.chunk;
    const int all = (most + BLOCK_TOKENS - 1) / BLOCK_TOKENS, end = all < b0 + a.chunk ? all : b0 + a.chunk;

    Running<HDP> run;
    run.clear();
    if constexpr (PAGED) {
        const int full = seq.len / BLOCK_TOKENS;  // full blocks hold codes
        const int* table = a.table + (size_t)seq.place * a.table_stride;
        Digits<HDP> qd;
        query_digits<HDP>(q, a.hd, a.scale, qd);
        int b = b0 + w;
        for (; b < end && b < full; b += WAVES) {
            const size_t at = (size_t)table[b] * a.kv_heads + g;
            const uint8_t* block = a.codes + at * (2 * BLOCK_TOKENS * HDP);
            const float2 sc = a.scales[at];
            if ((b + 1) * BLOCK_TOKENS <= least)
                codes_block<HDP, false>(block, sc, qd, 0, run);
            else
                codes_block<HDP, true>(block, sc, qd, seen - b * BLOCK_TOKENS, run);
        }
        if (b < end) {
            Pairs<HDP> qp;
            query_pairs<HDP>(q, a.hd, a.scale, qp);
            const _Float16* block = a.f16 + ((size_t)seq.place * a.kv_heads + g) * (2 * BLOCK_TOKENS * HDP);
            f16_block<HDP, true>(block, seq.len - b * BLOCK_TOKENS, qp, seen - b * BLOCK_TOKENS, run);
        }
    } else {
        Pairs<HDP> qp;
        query_pairs<HDP>(q, a.hd, a.scale, qp);
        const _Float16* states = a.f16 + ((size_t)seq.place * a.kv_heads + g) * a.blocks * (2 * BLOCK_TOKENS * HDP);
        for (int b = b0 + w; b < end; b += WAVES)
            f16_block<HDP, false>(states + (size_t)b * (2 * BLOCK_TOKENS * HDP), seq.len - b * BLOCK_TOKENS, qp,
                                  seq.len - b * BLOCK_TOKENS, run);
    }
    const float lsum = column_sum(run.l);
    if (lq == 0) {
        top[w][col] = run.m;
        sum[w][col] = lsum;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[w][col][16 * n + 4 * lq + r] = run.acc[n][r];
    __syncthreads();
    const int cols = min(columns - tile * 16, 16);
    // The sums of the waves' parts, relative to their largest score m.
    auto joined = [&](int cc, int e, float& m, float& l) {
        m = top[0][cc];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) m = __builtin_fmaxf(m, top[v][cc]);
        float o = 0.0f;
        l = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            // A wave that saw no key has sums of 0; NaN sums stay NaN.
            const float f = top[v][cc] == m ? 1.0f : __builtin_amdgcn_exp2f(top[v][cc] - m);
            o = __builtin_fmaf(part[v][cc][e], f, o);
            l = __builtin_fmaf(sum[v][cc], f, l);
        }
        return o;
    };
    auto store = [&](int cc, int e, float o, float l) {
        const int rr = (tile * 16 + cc) / a.group, hh = g * a.group + (tile * 16 + cc) % a.group;
        // No key at all: 0.
        if (e < a.hd) a.out[((size_t)(seq.first + rr) * a.kv_heads * a.group + hh) * a.hd + e] = l == 0.0f ? 0.0f : o / l;
    };
    if (seq.chunks == 1) {
        for (int i = t; i < cols * HDP; i += WAVES * WAVE) {
            float m, l;
            const float o = joined(i / HDP, i % HDP, m, l);
            store(i / HDP, i % HDP, o, l);
        }
        return;
    }
    for (int i = t; i < cols * HDP; i += WAVES * WAVE) {
        const int cc = i / HDP, e = i % HDP;
        float m, l;
        const float o = joined(cc, e, m, l);
        const size_t at = (size_t)blockIdx.x * 16 + cc;
        put(a.sums + at * HDP + e, o);
        if (e == 0) put(a.tops + at, (uint64_t)__float_as_uint(l) << 32 | __float_as_uint(m));
    }
    // Every store of the workgroup is in memory before its arrival is counted.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* counter = a.counters + seq.group + tile * a.kv_heads + g;
    if (t == 0) {
        const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        arrived = before + 1 == seq.chunks;
        if (before + 1 == seq.chunks) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!arrived) return;
    // Chunk v's item; wave w joins the chunks w, w + 4, .. of each column, lane l their elements 2 l, 2 l + 1.
    const size_t first = (size_t)seq.start + (size_t)tile * seq.chunks * a.kv_heads + g;
    for (int cc = 0; cc < cols; ++cc) {
        float m = -INFINITY, l = 0.0f;
        float2 o = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int v = w; v < seq.chunks; v += WAVES) {
            const size_t at = (first + (size_t)v * a.kv_heads) * 16 + cc;
            const float2 ml = get((const float*)(a.tops + at));
            const float2 x = 2 * lane < HDP ? get(a.sums + at * HDP + 2 * lane) : make_float2(0.0f, 0.0f);
            const float mn = __builtin_fmaxf(m, ml.x);
            const float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            const float h = ml.x == mn ? 1.0f : __builtin_amdgcn_exp2f(ml.x - mn);
            l = __builtin_fmaf(ml.y, h, l * f);
            o.x = __builtin_fmaf(x.x, h, o.x * f);
            o.y = __builtin_fmaf(x.y, h, o.y * f);
            m = mn;
        }
        if (lane == 0) {
            top[w][cc] = m;
            sum[w][cc] = l;
        }
        if (2 * lane < HDP) {
            part[w][cc][2 * lane] = o.x;
            part[w][cc][2 * lane + 1] = o.y;
        }
    }
    __syncthreads();
    for (int i = t; i < cols * HDP; i += WAVES * WAVE) {
        float m, l;
        const float o = joined(i / HDP, i % HDP, m, l);
        store(i / HDP, i % HDP, o, l);
    }
}

}  // namespace

// Items of one launch (a grid holds fewer than 2^32 threads), and the most
// where keys are split: what the scratch holds.
constexpr long long MOST_ITEMS = 1 << 23;
constexpr long long SPLIT_ITEMS = 1024;

void AttendScratch::make(int hdp, hipStream_t s) {
    memory.alloc(SPLIT_ITEMS * (16 * ((size_t)hdp * 4 + 8) + 4));
    // The counters are the last part.
    hipLaunchKernelGGL(clear_kernel, dim3(1), dim3(256), 0, s, (int*)((char*)memory.ptr + memory.bytes) - SPLIT_ITEMS,
                       (int)SPLIT_ITEMS);
    TRIT_HIP(hipGetLastError());
}

void attend(AttendArgs& a, const std::vector<AttendSeq>& seqs, bool paged, AttendScratch& scratch, hipStream_t s) {
    const int hdp = a.hd <= 64 ? 64 : 128;
    a.sums = scratch.memory.as<float>();
    a.tops = (uint64_t*)(a.sums + SPLIT_ITEMS * 16 * hdp);
    a.counters = (int*)(a.tops + SPLIT_ITEMS * 16);
    const auto tiles = [&](const AttendSeq& q) { return ((long long)q.rows * a.group + 15) / 16; };
    const auto blocks = [](const AttendSeq& q) { return (q.len + BLOCK_TOKENS - 1) / BLOCK_TOKENS; };
    for (size_t from = 0; from < seqs.size();) {
        // The launch's sequences, and its work in blocks of keys.
        long long whole = 0, work = 0;
        size_t to = from;
        for (a.n = 0; to < seqs.size() && a.n < CALL_SEQS; ++to) {
            if (seqs[to].rows == 0) continue;
            const long long items = tiles(seqs[to]) * a.kv_heads;
            if (items > MOST_ITEMS) fail("attention: more query rows than one launch takes");
            if (a.n && whole + items > MOST_ITEMS) break;
            whole += items;
            work += items * blocks(seqs[to]);
            a.s[a.n++] = seqs[to];
        }
        from = to;
        if (!a.n) return;
        // Chunks of as few blocks as keep the items within the scratch, a multiple of what the waves take at once.
        long long items = whole;
        a.chunk = INT_MAX / 2;
        if (whole < SPLIT_ITEMS) {
            const long long room = SPLIT_ITEMS - whole;
            a.chunk = (int)((work + room - 1) / room + WAVES - 1) / WAVES * WAVES;
            if (a.chunk < WAVES) a.chunk = WAVES;
        }
        items = 0;
        int groups = 0;
        for (int i = 0; i < a.n; ++i) {
            AttendSeq& q = a.s[i];
            const int nb = blocks(q);
            q.chunks = nb <= a.chunk ? 1 : (nb + a.chunk - 1) / a.chunk;
            q.start = (int)items;
            q.group = groups;
            items += tiles(q) * a.kv_heads * q.chunks;
            if (q.chunks > 1) groups += (int)tiles(q) * a.kv_heads;
        }
        const dim3 grid((unsigned)items), block(WAVES * WAVE);
        if (hdp == 64) {
            if (paged)
                hipLaunchKernelGGL((attend_kernel<64, true>), grid, block, 0, s, a);
            else
                hipLaunchKernelGGL((attend_kernel<64, false>), grid, block, 0, s, a);
        } else {
            if (paged)
                hipLaunchKernelGGL((attend_kernel<128, true>), grid, block, 0, s, a);
            else
                hipLaunchKernelGGL((attend_kernel<128, false>), grid, block, 0, s, a);
        }
        TRIT_HIP(hipGetLastError());
    }
}

}  // namespace trit
