// Attention of a few or many query rows to int8 blocks (a paged cache's full
// ones) and f16 blocks (its open ones, or an encoder's states).
#include <algorithm>
#include <climits>

#include "attend.h"
#include "blocks.h"
#include "device.h"

namespace trit {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
// Chunks that a tile's keys are split into at most.
constexpr int MOST_CHUNKS = 128;
// The largest fixed-point value of three int8 digits, and the factor that
// keeps the low part of an f16 pair clear of subnormal f16.
constexpr float FIXED = 8323072.0f;  // 127 * 65536
// What a product of the lowest digits starts from: its bits are a float's with
// the product added, so that it needs no conversion.
constexpr float LOWEST = 12582912.0f;  // 1.5 * 2^23
constexpr float PAIR = 1024.0f, LOG_PAIR = 10.0f;
// How far (in powers of two) scores may pass a softmax's reference: p * PAIR stays within f16.
constexpr float SLACK = 5.0f;

// The largest over a column's four lanes (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float column_max(float v) { return other_half_max(other_row_max(v)); }
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// The three digits of 4 fixed-point values (|x| <= FIXED), each digit's 4
// bytes in a word; the values come with CARRY added, which carries what a
// signed low digit takes from the next one. Flipping the low digits' top bits
// makes them signed; the highest one is.
constexpr int CARRY = 0x8080;
__device__ __forceinline__ void digits4(const uint32_t (&x)[4], int& d0, int& d1, int& d2) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    d0 = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
    d1 = (int)(__builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u);
    const uint32_t c = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(x[3], x[2], 0x0c0c0602u);
    d2 = (int)__builtin_amdgcn_perm(d, c, 0x05040100u);
}

// A wave's running softmax of 16 columns (query rows of the heads that share
// a key head): lane l holds column l % 16, and of the output the dims
// 16 n + 4 (l / 16) + r.
template <int HDP>
struct Running {
    float m = -INFINITY;  // the sums' reference, in powers of two: the largest score so far but for SLACK
    float l = 0.0f;       // this lane's part of the sum of 2^(score - m)
    float extra = 0.0f;   // what each of acc holds too much
    v4f acc[HDP / 16];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < HDP / 16; ++n) acc[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// Scores u * f (f >= 0 or NaN; of codes: (u - LOWEST) * f) of a block to
// probabilities of that block alone, p = 2^((u - max) f) <= 1, in place; then
// the running sums take the block's largest score as theirs. Returned: what
// scales the block's products (0 where the column sees none of it). A block's
// probabilities become fixed-point values or f16 pairs relative to its own
// maximum, so that a long tail of small ones next to one large one far away
// keeps its digits. mask (the same for the wave): `seen` of the block's tokens
// count, whatever the others hold.
template <int HDP, bool CODES>
__device__ __forceinline__ float block_softmax(float (&u)[16], float f, bool mask, int seen, Running<HDP>& run) {
    const int lq = (threadIdx.x % WAVE) / 16;
    if (mask) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (16 * (i / 4) + 4 * lq + i % 4 >= seen) u[i] = -INFINITY;
    }
    float top = u[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = __builtin_fmaxf(top, u[i]);
    top = column_max(top);
    const bool any = top > -INFINITY;
    const float scaled = top * f;
    const float mb = !any ? -INFINITY : CODES ? __builtin_fmaf(-LOWEST, f, scaled) : scaled;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        // Codes: what the rounding of the largest score lifts above 1 is 1, as digits need it. A NaN becomes 0, but
        // then f is NaN and with it what is returned. f16: the difference first, never above 0.
        if (CODES)
            u[i] = __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(__builtin_fmaf(u[i], f, -scaled)), 0.0f, 1.0f);
        else
            u[i] = __builtin_amdgcn_exp2f((u[i] - top) * f);
    }
    if (mask) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (16 * (i / 4) + 4 * lq + i % 4 >= seen) u[i] = 0.0f;
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += u[i];
    // The reference moves, and the sums with it, only when a score passes it by more than SLACK.
    if (__any(mb > run.m + SLACK)) {
        const float mn = __builtin_fmaxf(run.m, mb);
        const float before = mn == run.m ? 1.0f : __builtin_amdgcn_exp2f(run.m - mn);
        run.m = mn;
        run.l *= before;
        run.extra *= before;
#pragma unroll
        for (int n = 0; n < HDP / 16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) run.acc[n][r] *= before;
    }
    const float now = any ? __builtin_amdgcn_exp2f(mb - run.m) : 0.0f;
    run.l = __builtin_fmaf(now, sum, run.l);
    return now;
}

// The 16 columns' queries in shared memory, each part in its operand order (a
// wave's lane reads 16 bytes at 16 * lane of each 1 KB):
//  digits: fixed point round(q * FIXED / max|q|), three digits;
//  pairs: f16 values hi + lo of q * PAIR / max|q|;
//  top: max|q|, NaN for a query with a NaN or an infinity.
template <int HDP, bool DIGITS>
struct Queries {
    __align__(16) int8_t digits[3][DIGITS ? 16 * HDP : 16];
    __align__(16) _Float16 pairs[2][16 * HDP];
    float top[16];
};

// Thread 16 c + i of the workgroup takes HDP / 16 consecutive values of column
// c; q: its values, or any readable address with valid false. (Loads under a
// condition each would wait for each: 13 us of a 15 us launch.)
template <int HDP, bool DIGITS>
__device__ __forceinline__ void load_queries(const float* q, bool valid, bool aligned, int hd, float scale,
                                             float (&v)[HDP / 16]) {
    constexpr int E = HDP / 16;
    const int e0 = threadIdx.x % 16 * E;
    if (aligned) {  // head_dim a multiple of 4
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 x = gload_f4(q + (e0 + i < hd ? e0 + i : 0));
            v[i] = x.x;
            v[i + 1] = x.y;
            v[i + 2] = x.z;
            v[i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = *gmem(q + (e0 + i < hd ? e0 + i : 0));
    }
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = valid && e0 + i < hd ? v[i] * scale : 0.0f;
}
template <int HDP, bool DIGITS>
__device__ __forceinline__ void put_queries(const float (&v)[HDP / 16], bool pairs, Queries<HDP, DIGITS>& out) {
    constexpr int E = HDP / 16;
    const int col = threadIdx.x / 16, e0 = threadIdx.x % 16 * E;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) top = v[i] == v[i] ? __builtin_fmaxf(top, __builtin_fabsf(v[i])) : INFINITY;
    top = __builtin_fmaxf(top, dpp<DPP_XOR1>(top));
    top = __builtin_fmaxf(top, dpp<DPP_XOR2>(top));
    top = __builtin_fmaxf(top, dpp<DPP_HALF_MIRROR>(top));
    top = __builtin_fmaxf(top, dpp<DPP_MIRROR>(top));
    const bool finite = top < INFINITY;
    // Queries below 1e-30 have scores that differ by nothing.
    top = __builtin_fmaxf(top, 1e-30f);
    if (threadIdx.x % 16 == 0) out.top[col] = finite ? top : NAN;
    if (DIGITS) {
        const float inv = FIXED / top;
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            uint32_t x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = (uint32_t)((finite ? (int)__builtin_rintf(v[i + r] * inv) : 0) + CARRY);
            int d[3];
            digits4(x, d[0], d[1], d[2]);
            const int e = e0 + i, at = e / 64 * 1024 + (e % 64 / 16 * 16 + col) * 16 + e % 16;
#pragma unroll
            for (int j = 0; j < 3; ++j) *(int*)(out.digits[j] + at) = d[j];
        }
    }
    if (!pairs) return;
    const float inv = PAIR / top;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
        const int e = e0 + i, at = e / 32 * 512 + (e % 32 / 8 * 16 + col) * 8 + e % 8;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float x = finite ? v[i + r] * inv : 0.0f;
            const _Float16 hi = (_Float16)x;
            out.pairs[0][at + r] = hi;
            out.pairs[1][at + r] = (_Float16)(x - (float)hi);
        }
    }
}

// Values that are computed here. (The compiler otherwise moves the end of a
// product behind the branch around the next block's loads, where its integer
// parts and those loads' registers together spill, and a reload in the loop
// waits for every load.)
__device__ __forceinline__ void pin(v4f& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void pin(float& a, float& b, float& c, float& d) {
    asm volatile("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
}

// 16 bytes of a lane at a wave's address (in scalar registers) and the lane's offset.
__device__ __forceinline__ v4i load16(const uint8_t* wave, uint32_t lane) {
    return *(const TRIT_GLOBAL v4i*)((const TRIT_GLOBAL uint8_t*)wave + lane);
}

// The three digits' products as one number plus LOWEST. |c| <= 128 * 127 *
// 128, so the lowest one's stays within LOWEST's exponent and the others' sum
// within 32 bits. LOWEST is one and a half codes of the largest query value or
// probability, so it costs a sum no digit that counts; scores lose it with
// their largest, outputs at the end. (A conversion in its place: a prompt of
// 1564 rows after 1000 tokens 65 us, so 63.4; four of 1564 118, so 115.)
__device__ __forceinline__ float join_digits(int c0, int c1, int c2) {
    return __builtin_fmaf((float)((c2 << 8) + c1), 256.0f, __int_as_float(c0));
}
__device__ __forceinline__ v4i lowest() {
    const int x = __float_as_int(LOWEST);
    return v4i{x, x, x, x};
}

// A full block of int8 codes, its keys' and values' fragments in registers.
// Both products run in integers: the query and the probabilities are three
// int8 digits each, so their products with the codes are exact, and what is
// rounded is one fixed-point step of 24 bits.
template <int HDP>
__device__ __forceinline__ void codes_scores(const v4i (&kf)[HDP / 16], const v4i (&qd)[3][HDP / 64], float (&u)[16]) {
    constexpr int KS = HDP / 64;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        v4i c[3];
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            c[j] = j ? v4i{0, 0, 0, 0} : lowest();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                c[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t * KS + ks], qd[j][ks], c[j], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) u[4 * t + r] = join_digits(c[0][r], c[1][r], c[2][r]);
        pin(u[4 * t], u[4 * t + 1], u[4 * t + 2], u[4 * t + 3]);
    }
}
template <int HDP>
__device__ __forceinline__ void codes_values(const v4i (&vf)[HDP / 16], const float (&p)[16], float w,
                                             Running<HDP>& run) {
    v4i pd[3];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        uint32_t x[4];
        // round(p * FIXED) + CARRY in the low bits of a float of exponent 2^23: below 2^23 as p is at most 1.
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = __float_as_uint(__builtin_fmaf(p[4 * t + r], FIXED, 8388608.0f + CARRY));
        int d0, d1, d2;
        digits4(x, d0, d1, d2);
        pd[0][t] = d0;
        pd[1][t] = d1;
        pd[2][t] = d2;
    }
#pragma unroll
    for (int n = 0; n < HDP / 16; ++n) {
        v4i c[3];
#pragma unroll
        for (int j = 0; j < 3; ++j)
            c[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[n], pd[j], j ? v4i{0, 0, 0, 0} : lowest(), 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            run.acc[n][r] = __builtin_fmaf(join_digits(c[0][r], c[1][r], c[2][r]), w, run.acc[n][r]);
        pin(run.acc[n]);
    }
    run.extra = __builtin_fmaf(LOWEST, w, run.extra);
}

__device__ __forceinline__ bool any_nan(v8h x) {
    const v4i w = __builtin_bit_cast(v4i, x);
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) hit |= (((uint32_t)w[i] & 0x7fff7fffu) + 0x03ff03ffu) & 0x80008000u;
    return hit != 0;
}

__device__ __forceinline__ v8h load8h(const _Float16* wave, uint32_t lane) {
    return *(const TRIT_GLOBAL v8h*)((const TRIT_GLOBAL uint8_t*)wave + lane);
}

// An f16 block, the queries (from shared memory) and probabilities as f16 pairs.
template <int HDP>
__device__ __forceinline__ void f16_scores(const v8h (&kf)[HDP / 8], const _Float16* hi, const _Float16* lo,
                                           float (&u)[16]) {
    constexpr int KS = HDP / 32;
    const int lane = threadIdx.x % WAVE;
    v4f c[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const v8h qh = *(const v8h*)(hi + ks * 512 + lane * 8), ql = *(const v8h*)(lo + ks * 512 + lane * 8);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            c[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t * KS + ks], ql, c[t], 0, 0, 0);
            c[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t * KS + ks], qh, c[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        pin(c[t]);
#pragma unroll
        for (int r = 0; r < 4; ++r) u[4 * t + r] = c[t][r];
    }
}
__device__ __forceinline__ void value_pairs(const float (&p)[16], v8h (&ph)[2], v8h (&pl)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float x = p[i] * PAIR;
        const _Float16 hi = (_Float16)x;
        ph[i / 8][i % 8] = hi;
        pl[i / 8][i % 8] = (_Float16)(x - (float)hi);
    }
}
template <int HDP>
__device__ __forceinline__ void f16_values(const v8h (&vf)[HDP / 8], const float (&p)[16], float now,
                                           Running<HDP>& run) {
    v8h ph[2], pl[2];
    value_pairs(p, ph, pl);
    const float w = now * (1.0f / PAIR);
#pragma unroll
    for (int n = 0; n < HDP / 16; ++n) {
        v4f c = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[2 * n + s], pl[s], c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[2 * n + s], ph[s], c, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) run.acc[n][r] = __builtin_fmaf(c[r], w, run.acc[n][r]);
        pin(run.acc[n]);
    }
}

// A sequence's open block: values behind its last token are left from other
// sequences and taken as 0; a NaN among the valid ones counts for the columns
// that see its token and no others -- found by a product of its own.
template <int HDP>
__device__ __forceinline__ void open_values(v8h (&vf)[HDP / 8], const float (&p)[16], float now, int tokens, int seen,
                                            Running<HDP>& run) {
    constexpr int NT = HDP / 16;
    const int lq = (threadIdx.x % WAVE) / 16;
    bool nans = false;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        // The lane's tokens of this half that are valid, as a mask of its 8 halves.
        v4i keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 32 * s + 16 * (i / 2) + 4 * lq + 2 * (i % 2);
            keep[i] = t + 1 < tokens ? -1 : t < tokens ? 0xffff : 0;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            vf[2 * n + s] = __builtin_bit_cast(v8h, __builtin_bit_cast(v4i, vf[2 * n + s]) & keep);
            nans |= any_nan(vf[2 * n + s]);
        }
    }
    if (__any(nans)) {
        v8h sees[2];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sees[i / 8][i % 8] = (_Float16)(16 * (i / 4) + 4 * lq + i % 4 < min(seen, tokens) ? 1.0f : 0.0f);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            v4f count = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                v8h is;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const _Float16 x = vf[2 * n + s][i];
                    is[i] = (_Float16)(x != x ? 1.0f : 0.0f);
                    vf[2 * n + s][i] = x != x ? (_Float16)0.0f : x;
                }
                count = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, sees[s], count, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (count[r] > 0.0f) run.acc[n][r] = NAN;
        }
    }
    f16_values<HDP>(vf, p, now, run);
}

__global__ void clear_kernel(int* p, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) p[i] = 0;
}

// Words that other workgroups of the launch read: to and from memory past the
// caches that a reader on another XCD does not share.
__device__ __forceinline__ void put(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get(const float* p) {
    const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Block (item): sequence, key head g, TILES tiles of 16 columns (query row r,
// head g * group + c of it: column r * group + c) and a chunk of its key blocks
// (two tiles: all of them). Each tile's waves take the chunk's blocks in turn
// and join their sums in shared memory. Of the workgroups of a tile's chunks
// the last to end joins theirs, in the chunks' order.
template <int HDP, bool PAGED, int WAVES, int TILES = 1>
__global__ __launch_bounds__(WAVES* WAVE, 2) void attend_kernel(AttendArgs a) {
    constexpr int NT = HDP / 16, KS = HDP / 64, PS = HDP + 4;
    constexpr int KEYED = WAVES / TILES;  // waves that share a tile's keys
    constexpr size_t BLOCK = 2 * BLOCK_TOKENS * HDP;
    __shared__ Queries<HDP, PAGED> queries[TILES];
    __shared__ float top[WAVES][16], sum[WAVES][16];
    __shared__ __align__(16) float part[WAVES][16][PS];
    __shared__ bool arrived;
    const int t = threadIdx.x, lane = t % WAVE, col = lane % 16, lq = lane / 16;
    const int w = __builtin_amdgcn_readfirstlane(t / WAVE);
    // The last sequence whose items start at or before this one (the starts behind the last are past every item).
    const int g = blockIdx.x;
    int si = a.n == 1;
    if (!si)
#pragma unroll
        for (int i = 0; i < CALL_SEQS; i += WAVE) si += __popcll(__ballot(a.s[i + lane].start <= (int)blockIdx.y));
    const AttendSeq seq = a.s[si - 1];
    const int item = (int)blockIdx.y - seq.start;
    const int upto = seq.chunks == 1 ? item : item / seq.chunks, chunk = item - upto * seq.chunks;
    // The last rows' tiles first: they see the most.
    const int columns = seq.rows * a.group;
    const int tile = ((columns - 1) / (16 * TILES) - upto) * TILES, cols = min(columns - tile * 16, 16 * TILES);
    // The wave's tile of the workgroup's, its columns (none: 0 or less) and its turn at the tile's keys.
    const int mine = w / KEYED, turn = w % KEYED, own = min(cols - 16 * mine, 16);
    const Queries<HDP, PAGED>& qs = queries[mine];
    // Column c's row and head: row0 + (rest + c) / group. The quotient is of small whole numbers, exact in f32.
    const int row0 = tile * 16 / a.group, rest = tile * 16 - row0 * a.group;
    const float per = 1.0f / (float)a.group;
    auto row_of = [&](int c) { return (int)(((float)(rest + c) + 0.5f) * per); };

    // The thread's query values are on their way while the first keys are.
    float qv[TILES][NT];
    if (t < 256) {
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int c = 16 * i + t / 16, r = row_of(c), h = g * a.group + rest + c - r * a.group;
            const bool valid = c < cols;
            load_queries<HDP, PAGED>(valid ? a.q + (size_t)(seq.first + row0 + r) * a.qs + (size_t)h * a.hd : a.q, valid,
                                     a.aligned, a.hd, a.scale, qv[i]);
        }
    }
    // Keys the lane's column sees, and the wave's tile's most and least.
    const int ahead = PAGED ? seq.len - seq.rows + 1 + row0 : seq.len;
    const int least = PAGED ? ahead + (rest + 16 * mine) / a.group : ahead;
    const int most = own <= 0 ? 0 : PAGED ? ahead + (rest + 16 * mine + own - 1) / a.group : ahead;
    const int seen = PAGED ? ahead + row_of(16 * mine + min(col, max(own - 1, 0))) : ahead;
    const int b0 = chunk * a.chunk;
    // Whether any column of the workgroup meets f16 values.
    const int full = seq.len / BLOCK_TOKENS;  // full blocks hold codes
    const bool pairs =
        !PAGED || (full < b0 + a.chunk && ahead + (rest + cols - 1) / a.group > full * BLOCK_TOKENS);
    auto put_all = [&] {
        if (t < 256) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) put_queries<HDP, PAGED>(qv[i], pairs, queries[i]);
        }
        __syncthreads();
    };
    const int all = (most + BLOCK_TOKENS - 1) / BLOCK_TOKENS, end = all < b0 + a.chunk ? all : b0 + a.chunk;

    Running<HDP> run;
    run.clear();
    int b = b0 + turn;
    const uint32_t lane16 = lane * 16;
    if constexpr (PAGED) {
        const int last = end < full ? end : full;
        const int* table = a.table + (size_t)seq.place * a.table_stride;
        v4i kf[NT], vf[NT];
        float2 sc = make_float2(0.0f, 0.0f);
        int page = b < last ? table[b] : 0;
        const uint8_t* block = nullptr;
        if (b < last) {
            const size_t at = (size_t)page * a.kv_heads + g;
            block = a.codes + at * BLOCK;
            sc = a.scales[at];
#pragma unroll
            for (int i = 0; i < NT; ++i) kf[i] = load16(block + i * 1024, lane16);
#pragma unroll
            for (int i = 0; i < NT; ++i) vf[i] = load16(block + BLOCK / 2 + i * 1024, lane16);
            page = b + KEYED < last ? table[b + KEYED] : 0;
        }
        put_all();
        v4i qd[3][KS];
#pragma unroll
        for (int j = 0; j < 3; ++j)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qd[j][ks] = *(const v4i*)(qs.digits[j] + ks * 1024 + lane16);
        const float step = qs.top[col] * (LOG2E / FIXED);
        for (; b < last; b += KEYED) {
            float u[16];
            codes_scores<HDP>(kf, qd, u);
            const bool more = b + KEYED < last;
            const float2 s0 = sc;
            const uint8_t* next = block;
            if (more) {
                const size_t at = (size_t)page * a.kv_heads + g;
                next = a.codes + at * BLOCK;
                sc = a.scales[at];
                page = b + 2 * KEYED < last ? table[b + 2 * KEYED] : 0;
#pragma unroll
                for (int i = 0; i < NT; ++i) kf[i] = load16(next + i * 1024, lane16);
            }
            const float now =
                block_softmax<HDP, true>(u, step * s0.x, (b + 1) * BLOCK_TOKENS > least, seen - b * BLOCK_TOKENS, run);
            // A column that sees nothing of the block takes nothing of it, also where its scale is NaN.
            codes_values<HDP>(vf, u, now == 0.0f && seen <= b * BLOCK_TOKENS ? 0.0f : now * s0.y * (1.0f / FIXED), run);
            if (more) {
                block = next;
#pragma unroll
                for (int i = 0; i < NT; ++i) vf[i] = load16(block + BLOCK / 2 + i * 1024, lane16);
            }
        }
        if (b < end) {
            const _Float16* open = a.f16 + ((size_t)seq.place * a.kv_heads + g) * BLOCK;
            v8h k16[2 * NT], v16[2 * NT];
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) k16[i] = load8h(open + i * 512, lane16);
            float u[16];
            const int tokens = seq.len - b * BLOCK_TOKENS, sees = seen - b * BLOCK_TOKENS;
            f16_scores<HDP>(k16, qs.pairs[0], qs.pairs[1], u);
            // (With the values' loads before the scores' products the 128-wide kernel spills.)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) v16[i] = load8h(open + BLOCK / 2 + i * 512, lane16);
            const float now = block_softmax<HDP, false>(u, qs.top[col] * (LOG2E / PAIR), true, min(sees, tokens), run);
            open_values<HDP>(v16, u, now, tokens, sees, run);
        }
    } else {
        const _Float16* states =
            a.f16 + ((size_t)seq.place * a.kv_heads + g) * a.blocks * BLOCK;
        // 64 wide, the next block's values are on their way too; 128 wide they would not fit the registers.
        constexpr bool AHEAD = HDP == 64;
        v8h kf[2 * NT], vf[2 * NT];
        auto load = [&](v8h(&f)[2 * NT], int at, int half) {
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) f[i] = load8h(states + at * BLOCK + half * (BLOCK / 2) + i * 512, lane16);
        };
        if (b < end) {
            load(kf, b, 0);
            if (AHEAD) load(vf, b, 1);
        }
        put_all();
        const float step = qs.top[col] * (LOG2E / PAIR);
        for (; b < end; b += KEYED) {
            float u[16];
            f16_scores<HDP>(kf, qs.pairs[0], qs.pairs[1], u);
            if (!AHEAD) {
                __builtin_amdgcn_sched_barrier(0);
                load(vf, b, 1);
            }
            const bool more = b + KEYED < end;
            if (more && AHEAD) load(kf, b + KEYED, 0);
            const float now =
                block_softmax<HDP, false>(u, step, (b + 1) * BLOCK_TOKENS > seen, seen - b * BLOCK_TOKENS, run);
            f16_values<HDP>(vf, u, now, run);
            if (more && !AHEAD) load(kf, b + KEYED, 0);
            if (more && AHEAD) load(vf, b + KEYED, 1);
        }
    }
    const float lsum = column_sum(run.l);
    if (lq == 0) {
        top[w][col] = run.m;
        sum[w][col] = lsum;
    }
    if (col < own) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
            *(v4f*)(part[w][col] + 16 * n + 4 * lq) = PAGED ? run.acc[n] - run.extra : run.acc[n];
    }
    __syncthreads();
    // Four dims of a column: the sums of the waves' parts, relative to their largest score m.
    auto joined = [&](int cc, int e, float& m, float& l) {
        const int v0 = cc / 16 * KEYED, c = cc % 16;
        m = top[v0][c];
#pragma unroll
        for (int v = 1; v < KEYED; ++v) m = __builtin_fmaxf(m, top[v0 + v][c]);
        v4f o = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        l = 0.0f;
#pragma unroll
        for (int v = 0; v < KEYED; ++v) {
            // A wave that saw no key has sums of 0; NaN sums stay NaN.
            const float f = top[v0 + v][c] == m ? 1.0f : __builtin_amdgcn_exp2f(top[v0 + v][c] - m);
            const v4f x = *(const v4f*)(part[v0 + v][c] + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(x[i], f, o[i]);
            l = __builtin_fmaf(sum[v0 + v][c], f, l);
        }
        return o;
    };
    auto store = [&](int cc, int e, v4f o, float l) {
        const int r = row_of(cc), h = g * a.group + rest + cc - r * a.group;
        float* out = a.out + ((size_t)(seq.first + row0 + r) * a.kv_heads * a.group + h) * a.hd + e;
        // No key at all: 0.
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = l == 0.0f ? 0.0f : o[i] * inv;
        if (a.aligned_out) {
            if (e < a.hd) *(v4f*)out = o;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e + i < a.hd) out[i] = o[i];
        }
    };
    constexpr int QUADS = HDP / 4;
    if (TILES == 2 || seq.chunks == 1) {
        for (int i = t; i < cols * QUADS; i += WAVES * WAVE) {
            float m, l;
            const v4f o = joined(i / QUADS, i % QUADS * 4, m, l);
            store(i / QUADS, i % QUADS * 4, o, l);
        }
        return;
    }
    for (int i = t; i < cols * QUADS; i += WAVES * WAVE) {
        const int cc = i / QUADS, e = i % QUADS * 4;
        float m, l;
        const v4f o = joined(cc, e, m, l);
        const size_t at = ((size_t)(seq.part + item) * a.kv_heads + g) * 16 + cc;
        uint64_t* sums = (uint64_t*)(a.sums + at * HDP + e);
        put(sums, (uint64_t)__float_as_uint(o[1]) << 32 | __float_as_uint(o[0]));
        put(sums + 1, (uint64_t)__float_as_uint(o[3]) << 32 | __float_as_uint(o[2]));
        if (e == 0) put(a.tops + at, (uint64_t)__float_as_uint(l) << 32 | __float_as_uint(m));
    }
    // Every store of the workgroup is in memory before its arrival is counted: put() writes through the L2, so the
    // wait is enough. (A release fence also writes back whatever else the L2 holds: the 32 ragged requests 39.8 us,
    // without 32.2.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* counter = a.counters + (seq.group + upto) * a.kv_heads + g;
    if (t == 0) {
        const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        arrived = before + 1 == seq.chunks;
        if (before + 1 == seq.chunks) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!arrived) return;
    // The chunks' largest scores and sums, then their outputs: a thread four dims of a column, its loads all in flight.
    const size_t first = (size_t)(seq.part + upto * seq.chunks) * a.kv_heads + g;
    float* tops = &part[0][0][0];
    float* sums = tops + 16 * MOST_CHUNKS;
    static_assert(sizeof(part) >= 2 * 16 * MOST_CHUNKS * sizeof(float), "a chunk's entries fit the waves' parts");
    for (int i = t; i < cols * seq.chunks; i += WAVES * WAVE) {
        const int cc = i / seq.chunks, v = i - cc * seq.chunks;
        const float2 ml = get((const float*)(a.tops + (first + (size_t)v * a.kv_heads) * 16 + cc));
        tops[i] = ml.x;
        sums[i] = ml.y;
    }
    __syncthreads();
    for (int i = t; i < cols * QUADS; i += WAVES * WAVE) {
        const int cc = i / QUADS, e = i % QUADS * 4;
        const float* m = tops + cc * seq.chunks;
        float most = m[0];
        for (int v = 1; v < seq.chunks; ++v) most = __builtin_fmaxf(most, m[v]);
        float l = 0.0f;
        v4f o = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int v = 0; v < seq.chunks; ++v) {
            const float* at = a.sums + ((first + (size_t)v * a.kv_heads) * 16 + cc) * HDP + e;
            const float2 x = get(at), y = get(at + 2);
            const float f = m[v] == most ? 1.0f : __builtin_amdgcn_exp2f(m[v] - most);
            l = __builtin_fmaf(sums[cc * seq.chunks + v], f, l);
            o[0] = __builtin_fmaf(x.x, f, o[0]);
            o[1] = __builtin_fmaf(x.y, f, o[1]);
            o[2] = __builtin_fmaf(y.x, f, o[2]);
            o[3] = __builtin_fmaf(y.y, f, o[3]);
        }
        store(cc, e, o, l);
    }
}

// ---- many rows -------------------------------------------------------------

// The f16 pairs hi + lo of two values. (The factor -1 comes in a register the
// compiler does not know the value of: it makes one mixed-precision
// multiply-add of each rest, a conversion and a subtraction otherwise.)
__device__ __forceinline__ void split2(float a, float b, float minus_one, uint32_t& hi, uint32_t& lo) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 h = {(_Float16)a, (_Float16)b};
    uint32_t bits = __builtin_bit_cast(uint32_t, h);
    asm("" : "+v"(bits));
    h = __builtin_bit_cast(h2, bits);
    const h2 l = {(_Float16)__builtin_fmaf((float)h[0], minus_one, a), (_Float16)__builtin_fmaf((float)h[1], minus_one, b)};
    hi = bits;
    lo = __builtin_bit_cast(uint32_t, l);
}

// Attention to states where a slot is asked by many query columns: workgroup
// (g, item) takes 64 columns of a slot (column r * group + c: row r, head
// g * group + c), a wave 16 of them over every key block. The blocks pass
// through shared memory, once for the four waves, the next one's loads in
// flight while one is worked on. What binds is the issue of vector and matrix
// instructions together: about 150 and 32 a block and wave (64 wide), the sum
// of their cycles near the time the compute units are busy. (32 columns a
// wave read each fragment once for two tiles, but leave half the waves: 63 us
// for 448 rows over each of 8 audios where this takes 55.)
//
// A probability is an f16 pair relative to a reference within SLACK of the
// running maximum, times PAIR; what a pair loses is below 2^-34 of the
// largest, so sums run on across blocks.
template <int HDP>
__global__ __launch_bounds__(256, HDP == 64 ? 4 : 2) void attend_rows_kernel(AttendArgs a) {
    constexpr int NT = HDP / 16, KS = HDP / 32, F = BLOCK_TOKENS * HDP * 2 / 8 / 256;  // 16-byte pieces a thread
    constexpr size_t BLOCK = 2 * BLOCK_TOKENS * HDP;
    __shared__ __align__(16) _Float16 kv[BLOCK];
    const int t = threadIdx.x, lane = t % WAVE, col = lane % 16, lq = lane / 16;
    const int w = __builtin_amdgcn_readfirstlane(t / WAVE);
    const int g = blockIdx.x;
    int si = a.n == 1;
    if (!si)
#pragma unroll
        for (int i = 0; i < CALL_SEQS; i += WAVE) si += __popcll(__ballot(a.s[i + lane].start <= (int)blockIdx.y));
    const AttendSeq seq = a.s[si - 1];
    const int columns = seq.rows * a.group;
    const int tile = ((int)blockIdx.y - seq.start) * 4 + w;  // the wave's
    const bool idle = tile * 16 >= columns;  // a wave without columns: it moves blocks only
    const int end = (seq.len + BLOCK_TOKENS - 1) / BLOCK_TOKENS;
    const _Float16* states = a.f16 + ((size_t)seq.place * a.kv_heads + g) * a.blocks * BLOCK;

    uint4 piece[F];  // the thread's pieces of the next block
    auto fetch = [&](int b) {
#pragma unroll
        for (int i = 0; i < F; ++i) piece[i] = gload_u4(states + b * BLOCK + i * 2048 + t * 8);
    };
    if (end > 0) fetch(0);
    // The lane's column: row and head.
    const int row0 = tile * 16 / a.group, x0 = tile * 16 - row0 * a.group + col;
    const int r = (int)(((float)x0 + 0.5f) * (1.0f / (float)a.group)), row = row0 + r, head = g * a.group + x0 - r * a.group;
    const bool valid = tile * 16 + col < columns;
    // Its query values: dims 32 ks + 8 lq + i, as f16 pairs.
    v8h qh[KS], ql[KS];
    float step;
    {
        const float* q = valid ? a.q + (size_t)(seq.first + row) * a.qs + (size_t)head * a.hd : a.q;
        float v[KS][8], top = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int e = 32 * ks + 8 * lq;
            if (a.aligned) {
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 x = gload_f4(q + (e + i < a.hd ? e + i : 0));
                    v[ks][i] = x.x;
                    v[ks][i + 1] = x.y;
                    v[ks][i + 2] = x.z;
                    v[ks][i + 3] = x.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[ks][i] = *gmem(q + (e + i < a.hd ? e + i : 0));
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = valid && 32 * ks + 8 * lq + i < a.hd ? v[ks][i] * a.scale : 0.0f;
                v[ks][i] = x;
                top = x == x ? __builtin_fmaxf(top, __builtin_fabsf(x)) : INFINITY;
            }
        top = column_max(top);
        const bool finite = top < INFINITY;
        top = __builtin_fmaxf(top, 1e-30f);
        const float inv = PAIR / top;
        step = finite ? top * (LOG2E / PAIR) : NAN;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = finite ? v[ks][i] * inv : 0.0f;
                qh[ks][i] = (_Float16)x;
                ql[ks][i] = (_Float16)(x - (float)qh[ks][i]);
            }
    }
    float minus_one = -1.0f;
    asm("" : "+v"(minus_one));
    float m = -INFINITY, l = 0.0f;  // m: the reference of the sums
    v4f acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    for (int b = 0; b < end; ++b) {
#pragma unroll
        for (int i = 0; i < F; ++i) *(uint4*)(kv + i * 2048 + t * 8) = piece[i];
        __syncthreads();
        if (b + 1 < end) fetch(b + 1);
        if (!idle) {
            const _Float16* k = kv + lane * 8;
            v4f u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v8h kf = *(const v8h*)(k + (i * KS + ks) * 512);
                    u[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[ks], u[i], 0, 0, 0);
                    u[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[ks], u[i], 0, 0, 0);
                }
            const int tokens = seq.len - b * BLOCK_TOKENS;
            const bool mask = tokens < BLOCK_TOKENS;
            v8h ph[2], pl[2];
            if (mask) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (16 * (i / 4) + 4 * lq + i % 4 >= tokens) u[i / 4][i % 4] = -INFINITY;
            }
            float top = u[0][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = __builtin_fmaxf(top, u[i / 4][i % 4]);
            top = column_max(top) * step;
            if (__any(top > m + SLACK)) {
                const float mn = __builtin_fmaxf(m, top);
                const float before = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= before;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][i] *= before;
            }
            const float ref = (m > -INFINITY ? m : 0.0f) - LOG_PAIR;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float p = __builtin_amdgcn_exp2f(__builtin_fmaf(u[i / 4][i % 4], step, -ref));
                u[i / 4][i % 4] = p;
                sum += p;
            }
            l += sum;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                v4i hi, lo;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t x, y;
                    split2(u[2 * s + i / 2][2 * i % 4], u[2 * s + i / 2][2 * i % 4 + 1], minus_one, x, y);
                    hi[i] = (int)x;
                    lo[i] = (int)y;
                }
                ph[s] = __builtin_bit_cast(v8h, hi);
                pl[s] = __builtin_bit_cast(v8h, lo);
            }
            const _Float16* v = kv + BLOCK / 2 + lane * 8;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const v8h vf = *(const v8h*)(v + (2 * n + s) * 512);
                    acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[s], acc[n], 0, 0, 0);
                    acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[s], acc[n], 0, 0, 0);
                }
        }
        __syncthreads();  // the block is read
    }
    l = column_sum(l);
    if (!valid) return;
    // No key at all: 0.
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float* out = a.out + ((size_t)(seq.first + row) * a.kv_heads * a.group + head) * a.hd;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 16 * n + 4 * lq + i;
            if (e < a.hd) out[e] = l == 0.0f ? 0.0f : acc[n][i] * inv;
        }
}

}  // namespace

// Tiles of one launch (the grid's second dimension), and the most workgroups
// of split keys: what the scratch holds.
constexpr long long MOST_TILES = 50000;
constexpr long long SPLIT_ITEMS = 1024;
// Workgroups of 8 waves that the compute units take at once.
constexpr long long FEW_ITEMS = 256;
// The least workgroups of two tiles that a paged launch takes, where nine
// tenths of the second ones are there (60 requests of a single tile, 20 heads
// of 64, 29 us with one, 34 with room for two): a wave's keys are twice as
// many, so its fixed part (queries, first loads, join) weighs half. 16/8 heads
// of 128, us with one tile and with two: 3000 rows after 1000 tokens (1500 such
// workgroups) 137 and 129, two prompts of 1564 (1568) 66 and 59, four (3136)
// 126 and 111; 1564 rows after 1000 (784) 60.3 and 60.9, 512 after 512 (256)
// 13.2 and 18.3. 20 heads of 64: 1880 103 and 101, 3920 90 and 80; 640 27 and
// 30.
constexpr long long PAIR_ITEMS = 1024;
// Columns of a key head from which the many-row kernel takes a slot, and the
// least workgroups it takes: with fewer its serial pass over the blocks is the
// longer one. 64 wide, 20 heads, us here and on attend_kernel: 320 workgroups
// 47 and 37, 500 57 and 68, 2000 120 and 165; 128 wide: 256 54 and 53, 392 92
// and 102, 1568 186 and 235. (The same form for a paged cache, codes widened
// into shared memory, was no shorter than attend_kernel: 1564 rows after 1000
// tokens 102 and 61.)
constexpr long long MANY_COLUMNS = 64, MANY_ITEMS = 384;

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
    a.aligned = a.hd % 4 == 0 && a.qs % 4 == 0 && (uintptr_t)a.q % 16 == 0;
    a.aligned_out = a.hd % 4 == 0 && (uintptr_t)a.out % 16 == 0;
    // Slots that many columns ask, in launches of their own.
    std::vector<AttendSeq> few, many;
    const auto wide = [&](const AttendSeq& q) { return ((long long)q.rows * a.group + 63) / 64; };
    long long wides = 0;
    for (const AttendSeq& q : seqs) {
        if (!q.rows) continue;
        if (tiles(q) > MOST_TILES) fail("attention: more query rows than one launch takes");
        const bool is = !paged && (long long)q.rows * a.group >= MANY_COLUMNS;
        if (is) wides += wide(q);
        (is ? many : few).push_back(q);
    }
    if (wides * a.kv_heads < MANY_ITEMS) {
        few.insert(few.end(), many.begin(), many.end());
        many.clear();
    }
    // The longest first, so that the last workgroups are short.
    std::stable_sort(many.begin(), many.end(), [](const AttendSeq& x, const AttendSeq& y) { return x.len > y.len; });
    for (size_t at = 0; at < many.size();) {
        long long items = 0;
        for (a.n = 0; at < many.size() && a.n < CALL_SEQS; ++at) {
            AttendSeq q = many[at];
            if (a.n && items + wide(q) > MOST_TILES) break;
            q.start = (int)items;
            items += wide(q);
            a.s[a.n++] = q;
        }
        for (int i = a.n; i < CALL_SEQS; ++i) a.s[i].start = INT_MAX;
        auto kernel = hdp == 64 ? attend_rows_kernel<64> : attend_rows_kernel<128>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.kv_heads, (unsigned)items), dim3(256), 0, s, a);
        TRIT_HIP(hipGetLastError());
    }
    for (size_t from = 0; from < few.size();) {
        // The launch's sequences, and its work in blocks of keys.
        long long whole = 0, work = 0;
        int most = 0;
        size_t to = from;
        for (a.n = 0; to < few.size() && a.n < CALL_SEQS; ++to) {
            if (a.n && whole + tiles(few[to]) > MOST_TILES) break;
            whole += tiles(few[to]);
            work += tiles(few[to]) * blocks(few[to]);
            most = std::max(most, blocks(few[to]));
            a.s[a.n++] = few[to];
        }
        from = to;
        if (!a.n) return;
        // Where 8-wave workgroups leave compute units free, latency is what counts: 8 waves with two rounds and no
        // join up to 16 blocks, one round a chunk above. One token of 700, 16/8 heads of 128: 8.1 us (4 waves a
        // chunk: 8.4); 5 rows over 1500 states, 20 heads of 64: 8.0 (8.8). Else 4 waves, and chunks of two rounds
        // or more: as few as make no more than two workgroups a compute unit, which is what they hold, or a quarter
        // more than there are without a split. 32 requests of 100 to 8001 tokens: 33.1 us with 512 workgroups,
        // 35.3 with 760, 41 with 2030; two of 131 K 101 us with 512, 105 with 1024, 112 with 8 waves.
        long long small = 0;
        for (int i = 0; i < a.n; ++i) {
            const long long nb = blocks(a.s[i]);
            small += tiles(a.s[i]) * (nb <= 16 ? 1 : (nb + 7) / 8);
        }
        const int waves = small * a.kv_heads <= FEW_ITEMS ? 8 : 4;
        long long split = 0;  // items of split sequences
        const auto items_of = [&](int chunk) {
            long long all = split = 0;
            for (int i = 0; i < a.n; ++i) {
                const long long c = std::max((blocks(a.s[i]) + chunk - 1) / chunk, 1), t = tiles(a.s[i]) * c;
                all += t;
                if (c > 1) split += t;
            }
            return all;
        };
        if (waves == 8) {
            a.chunk = std::max(most <= 16 ? 16 : 8, (most + MOST_CHUNKS - 1) / MOST_CHUNKS);
            items_of(a.chunk);
        } else {
            const long long room = std::max(2 * FEW_ITEMS / a.kv_heads, whole + whole / 4);
            a.chunk = (int)std::max({work / room, (long long)(most + MOST_CHUNKS - 1) / MOST_CHUNKS, 2LL * waves});
            a.chunk = (a.chunk + waves - 1) / waves * waves;
            while (items_of(a.chunk) > room || split * a.kv_heads > SPLIT_ITEMS)
                a.chunk += (a.chunk / 8 + waves) / waves * waves;
        }
        long long two = 0;
        for (int i = 0; i < a.n; ++i) two += (tiles(a.s[i]) + 1) / 2;
        const bool pairs = paged && !split && two * a.kv_heads >= PAIR_ITEMS && 5 * whole >= 9 * two;
        int items = 0, groups = 0, parts = 0;
        for (int i = 0; i < CALL_SEQS; ++i) {
            AttendSeq& q = a.s[i];
            if (i >= a.n) {
                q.start = INT_MAX;
                continue;
            }
            q.chunks = std::max((blocks(q) + a.chunk - 1) / a.chunk, 1);
            q.start = items;
            q.group = groups;
            q.part = parts;
            items += pairs ? (int)((tiles(q) + 1) / 2) : (int)tiles(q) * q.chunks;
            if (q.chunks > 1) {
                groups += (int)tiles(q);
                parts += (int)tiles(q) * q.chunks;
            }
        }
        const dim3 grid((unsigned)a.kv_heads, (unsigned)items), block((unsigned)(waves * WAVE));
        auto kernel = hdp == 64 ? (paged ? (waves == 4 ? attend_kernel<64, true, 4> : attend_kernel<64, true, 8>)
                                         : (waves == 4 ? attend_kernel<64, false, 4> : attend_kernel<64, false, 8>))
                                : (paged ? (waves == 4 ? attend_kernel<128, true, 4> : attend_kernel<128, true, 8>)
                                         : (waves == 4 ? attend_kernel<128, false, 4> : attend_kernel<128, false, 8>));
        if (pairs) kernel = hdp == 64 ? attend_kernel<64, true, 4, 2> : attend_kernel<128, true, 4, 2>;
        hipLaunchKernelGGL(kernel, grid, block, 0, s, a);
        TRIT_HIP(hipGetLastError());
    }
}

}  // namespace trit
