// A paged key/value cache of many sequences (include/trit_hip.h): full blocks
// of 64 tokens as int8 codes with a scale for each block and head, the open
// block of each sequence as f16.
#include <algorithm>
#include <cstring>
#include <mutex>

#include "../../include/trit_hip.h"
#include "attend.h"
#include "blocks.h"
#include "device.h"
#include "internal.h"
#include "page_book.h"

namespace trit {
namespace {

static_assert(PageBook::BLOCK == BLOCK_TOKENS, "one block size");

constexpr int THREADS = BLOCK_THREADS;
// Entries of one launch (kernel arguments).
constexpr int CALL_ENTRIES = 256;

// ---- device side -----------------------------------------------------------

// A layer's arrays. codes: by page and head, K then V, 64 * HDP bytes each in
// k8_at / v8_at order; scales: their two; open: by row and head, K then V,
// 64 * HDP halves each in k16_at / v16_at order (0 past head_dim).
struct Pool {
    uint8_t* codes;
    float2* scales;
    _Float16* open;
    int* table;
    int pages;  // the table's row length
    int kv_heads, hd;
};

struct RowsSeq {
    int row;    // of the table and the open blocks
    int len;    // tokens before the call (append), or in all (read)
    int at;     // the first token to read
    int count;  // rows of the call
    int first;  // its first one in the caller's arrays
};
struct RowsArgs {
    RowsSeq s[CALL_SEQS];
};

// Appends rows: workgroup (x, g, 2 i + V) writes keys (V 0) or values (1) of
// head g into the x-th block that sequence i's new rows touch -- as codes
// where the block becomes full, else as f16 into the open block. The first
// block's workgroup also writes the last, open one, after its own: it alone
// reads the open block's old rows, which the last block replaces.
//
// A code is round(127 h / a), halves to even: h times the rounded 127 / a
// rounds to it but within 8e-6 of a half (2^-24 of a quotient up to 127), and
// lanes that meet a value within 4e-5 divide: 127 h is exact, and no quotient
// of two f16 values rounds onto a half it is not. 60 sequences whose blocks
// become full, 8 heads of 128 (16 MB in, 8 out): 12.7 us, a division each
// 13.6; the same where none does: 4.4 us. Eight prompts of 37 to 1564 rows
// (42 MB in, 10 out): 13 us.
template <int HDP, bool V>
__device__ __forceinline__ void append_block(const Pool& p, const RowsSeq& s, const float* rows, long long stride,
                                             bool aligned, uint32_t* codes, uint32_t* red) {
    constexpr int G = BlockShare<HDP>::GROUPS, VALUES = BlockShare<HDP>::VALUES;
    constexpr uint32_t FINITE = 0x7f800000u;
    const int g = blockIdx.y, t = threadIdx.x, x = blockIdx.x;
    const int b0 = s.len / BLOCK_TOKENS, have = s.len % BLOCK_TOKENS;
    const int touched = (have + s.count + BLOCK_TOKENS - 1) / BLOCK_TOKENS;  // blocks
    const bool ends_full = (have + s.count) % BLOCK_TOKENS == 0;
    _Float16* open = p.open + (((size_t)s.row * p.kv_heads + g) * 2 + V) * (BLOCK_TOKENS * HDP);
    if (x + 1 < touched || ends_full) {
        const size_t page = (size_t)p.table[(size_t)s.row * p.pages + b0 + x] * p.kv_heads + g;
        float h[VALUES];
        load_share<HDP, V>(rows, stride, x * BLOCK_TOKENS - have, s.count, p.hd, aligned, h);
#pragma unroll
        for (int i = 0; i < VALUES; ++i) h[i] = (float)(_Float16)h[i];
        if (x == 0 && have) {
            // The tokens that the open block holds.
            uint2 old[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                int tok, e;
                share_at<HDP, V>(i, tok, e);
                old[i] = gload_u2(open + half_at<HDP, V>(tok, e));
            }
#pragma unroll
            for (int i = 0; i < G; ++i) {
                int tok, e;
                share_at<HDP, V>(i, tok, e);
                _Float16 o[4];
                __builtin_memcpy(o, &old[i], 8);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (tok + (V ? j : 0) < have) h[4 * i + j] = (float)o[j];
            }
        }
        if (p.hd < HDP) {
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                int tok, e;
                share_at<HDP, V>(i / 4, tok, e);
                if ((V ? e : e + i % 4) >= p.hd) h[i] = 0.0f;
            }
        }
        // The largest magnitude, by its bits: those of infinities and NaN are larger than any other's.
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) most = max(most, __float_as_uint(h[i]) & 0x7fffffffu);
        // (Below infinity magnitudes and their bits are in one order; from there on only "not finite" counts.)
        const bool odd = __any(most >= FINITE);
        const float wave = wave_max(__uint_as_float(most < FINITE ? most : 0));
        if (t % WAVE == 0) red[t / WAVE] = odd ? FINITE : __float_as_uint(wave);
        __syncthreads();
        most = red[0];
#pragma unroll
        for (int w = 1; w < THREADS / WAVE; ++w) most = max(most, red[w]);
        const bool bad = most >= FINITE;
        const float top = bad ? 0.0f : __uint_as_float(most);
        // round(h c) in the low bits of a float of exponent 2^23.
        constexpr float MAGIC = 12582912.0f;
        const float c = top > 0.0f ? 127.0f / top : 0.0f;
        float y[VALUES], near = 0.0f;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            h[i] = bad ? 0.0f : h[i];
            y[i] = __builtin_fmaf(h[i], c, MAGIC);
            near = __builtin_fmaxf(near, __builtin_fabsf(__builtin_fmaf(h[i], c, MAGIC - y[i])));
        }
        if (near > 0.49996f) {
#pragma unroll
            for (int i = 0; i < VALUES; ++i) y[i] = 127.0f * h[i] / top + MAGIC;
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            int tok, e;
            share_at<HDP, V>(i, tok, e);
            const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(y[4 * i + 1]), __float_as_uint(y[4 * i]), 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(y[4 * i + 3]), __float_as_uint(y[4 * i + 2]), 0x0c0c0400u);
            codes[code_at<HDP, V>(tok, e) / 4] = lo | hi << 16;
        }
        __syncthreads();
        uint4* dst = (uint4*)(p.codes + (page * 2 + V) * (BLOCK_TOKENS * HDP));
#pragma unroll
        for (int i = 0; i < BLOCK_TOKENS * HDP / 16; i += THREADS) dst[i + t] = *(const uint4*)(codes + (i + t) * 4);
        if (t == 0) (V ? p.scales[page].y : p.scales[page].x) = bad ? NAN : top / 127.0f;
    }
    // The open block at the end: its own workgroup is the first block's.
    if (x != 0 || ends_full) return;
    const int first = (touched - 1) * BLOCK_TOKENS - have, from = max(-first, 0), to = (have + s.count) % BLOCK_TOKENS;
    if (to - from <= 2) {
        // A step's one or two rows: a value a thread.
        const int tok = from + t / HDP, e = t % HDP;
        if (tok < to && e < p.hd) open[half_at<HDP, V>(tok, e)] = held(rows[(size_t)(first + tok) * stride + e]);
        return;
    }
    float h[VALUES];
    load_share<HDP, V>(rows, stride, first, s.count, p.hd, aligned, h);
    __syncthreads();  // the old rows are read
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
        int tok, e;
        share_at<HDP, V>(i / 4, tok, e);
        tok += V ? i % 4 : 0;
        e += V ? 0 : i % 4;
        if (tok >= from && tok < to && e < p.hd) open[half_at<HDP, V>(tok, e)] = held(h[i]);
    }
}
template <int HDP>
__global__ __launch_bounds__(THREADS) void append_kernel(Pool p, RowsArgs a, const float* k, long long ks,
                                                         const float* v, long long vs, bool aligned) {
    __shared__ __align__(16) uint32_t codes[BLOCK_TOKENS * HDP / 4];
    __shared__ uint32_t red[THREADS / WAVE];
    const RowsSeq s = a.s[blockIdx.z / 2];
    if (s.count == 0 || (int)blockIdx.x >= (s.len % BLOCK_TOKENS + s.count + BLOCK_TOKENS - 1) / BLOCK_TOKENS) return;
    const size_t column = (size_t)blockIdx.y * p.hd;
    if (blockIdx.z % 2)
        append_block<HDP, true>(p, s, v + (size_t)s.first * vs + column, vs, aligned, codes, red);
    else
        append_block<HDP, false>(p, s, k + (size_t)s.first * ks + column, ks, aligned, codes, red);
}

// Reads rows as the values they stand for: workgroup (x, g, 2 i + which), the
// x-th block that sequence i's range touches.
template <int HDP>
__global__ __launch_bounds__(THREADS) void read_kernel(Pool p, RowsArgs a, float* k, long long ks, float* v,
                                                       long long vs, bool aligned) {
    const bool which = blockIdx.z % 2;
    const int g = blockIdx.y, t = threadIdx.x;
    const RowsSeq s = a.s[blockIdx.z / 2];
    const int b = s.at / BLOCK_TOKENS + (int)blockIdx.x;
    const int from = max(s.at - b * BLOCK_TOKENS, 0), to = min(s.at + s.count - b * BLOCK_TOKENS, BLOCK_TOKENS);
    if (from >= to) return;
    float* out = which ? v : k;
    const long long stride = which ? vs : ks;
    const bool full = (b + 1) * BLOCK_TOKENS <= s.len;
    const int lane = t % WAVE, col = lane % 16, lq = lane / 16;
    float* rows = out + (s.first + (long long)b * BLOCK_TOKENS - s.at) * stride + (size_t)g * p.hd;
    auto store = [&](int tok, int e, float x) {
        if (tok >= from && tok < to && e < p.hd) rows[(size_t)tok * stride + e] = x;
    };
    // Four consecutive dims of a token.
    auto store4 = [&](int tok, int e, float a0, float a1, float a2, float a3) {
        if (aligned) {
            if (tok >= from && tok < to && e < p.hd) *(float4*)(rows + (size_t)tok * stride + e) = make_float4(a0, a1, a2, a3);
        } else {
            store(tok, e, a0);
            store(tok, e + 1, a1);
            store(tok, e + 2, a2);
            store(tok, e + 3, a3);
        }
    };
    // A wave takes whole 1 KB fragments, 16 bytes a lane, all on their way before the first is used.
    if (full) {
        constexpr int N = BLOCK_TOKENS * HDP / 16 / THREADS;
        const size_t page = (size_t)p.table[(size_t)s.row * p.pages + b] * p.kv_heads + g;
        const uint8_t* codes = p.codes + (page * 2 + which) * (BLOCK_TOKENS * HDP);
        const float scale = which ? p.scales[page].y : p.scales[page].x;
        uint4 c[N];
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = gload_u4(codes + (i * THREADS + t) * 16);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int f = (i * THREADS + t) / WAVE;
            const uint32_t words[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = (float)(int8_t)(words[j] >> (8 * r)) * scale;
                if (which) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) store(16 * j + 4 * lq + r, 16 * f + col, x[r]);
                } else {
                    constexpr int KS = HDP / 64;
                    store4(f / KS * 16 + col, f % KS * 64 + 16 * lq + 4 * j, x[0], x[1], x[2], x[3]);
                }
            }
        }
        return;
    }
    constexpr int N = BLOCK_TOKENS * HDP / 8 / THREADS;
    const _Float16* open = p.open + (((size_t)s.row * p.kv_heads + g) * 2 + which) * (BLOCK_TOKENS * HDP);
    // Only the fragments that hold wanted tokens: of K a tile of 16 tokens, of V 32.
    auto wanted = [&](int i) {
        const int f = (i * THREADS + t) / WAVE, first = which ? f % 2 * 32 : f / (HDP / 32) * 16;
        return first < to && first + (which ? 32 : 16) > from;
    };
    uint4 c[N];
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = gload_u4(open + (wanted(i) ? (i * THREADS + t) * 8 : lane * 8));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int f = (i * THREADS + t) / WAVE;
        _Float16 x[8];
        __builtin_memcpy(x, &c[i], 16);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (which) {
#pragma unroll
                for (int r = 0; r < 4; ++r) store(f % 2 * 32 + 16 * j + 4 * lq + r, f / 2 * 16 + col, (float)x[4 * j + r]);
            } else {
                constexpr int KS = HDP / 32;
                store4(f / KS * 16 + col, f % KS * 32 + 8 * lq + 4 * j, (float)x[4 * j], (float)x[4 * j + 1],
                       (float)x[4 * j + 2], (float)x[4 * j + 3]);
            }
        }
    }
}

struct TableArgs {
    PageBook::Entry e[CALL_ENTRIES];
};
__global__ void table_kernel(int* table, int pages, TableArgs a, int n) {
    const int i = threadIdx.x;
    if (i < n) table[(size_t)a.e[i].row * pages + a.e[i].block] = a.e[i].page;
}

// Open blocks and table rows from one row to another, of every layer:
// workgroup (copy, layer and head, quarter of the block).
struct CopyArgs {
    PageBook::RowCopy c[CALL_ENTRIES];
};
template <int HDP>
__global__ __launch_bounds__(THREADS) void row_kernel(const _Float16* from, int from_rows, _Float16* to, int to_rows,
                                                      int kv_heads, int* table, int pages, CopyArgs a) {
    const PageBook::RowCopy c = a.c[blockIdx.x];
    const int layer = blockIdx.y / kv_heads, g = blockIdx.y % kv_heads, t = threadIdx.x;
    if (blockIdx.y == 0 && blockIdx.z == 0)
        for (int i = t; i < c.blocks; i += THREADS)
            table[(size_t)c.dst * pages + i] = table[(size_t)c.src * pages + i];
    const int tokens = c.len % BLOCK_TOKENS;
    if (!tokens) return;
    // The 1 KB fragments that hold its tokens: of K whole tiles of 16, of V halves of 32.
    constexpr size_t BLOCK = 2 * BLOCK_TOKENS * HDP;
    constexpr int N = BLOCK / 8 / THREADS / 4, KF = 4 * (HDP / 32);
    const _Float16* src = from + (((size_t)layer * from_rows + c.src) * kv_heads + g) * BLOCK;
    _Float16* dst = to + (((size_t)layer * to_rows + c.dst) * kv_heads + g) * BLOCK;
    uint4 x[N];
    bool needed[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int u = (blockIdx.z * N + i) * THREADS + t, f = u / WAVE;
        needed[i] = f < KF ? f / (HDP / 32) * 16 < tokens : (f - KF) % 2 * 32 < tokens;
        if (needed[i]) x[i] = gload_u4(src + u * 8);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (needed[i]) *(uint4*)(dst + ((blockIdx.z * N + i) * THREADS + t) * 8) = x[i];
}

// Pages from one pool to another (or within one: no page is both read and
// written), of every layer: workgroup (move, layer and head); and entries of
// the destination's table.
constexpr int CALL_MOVES = 128;
struct MoveArgs {
    PageBook::PageMove m[CALL_MOVES];
    PageBook::Entry e[CALL_MOVES];
    int entries;  // of e, written by the workgroup of move 0, layer 0 and head 0
};
template <int HDP>
__global__ __launch_bounds__(THREADS) void page_kernel(const uint8_t* codes, const float2* scales, int pages,
                                                       uint8_t* to_codes, float2* to_scales, int to_pages,
                                                       int kv_heads, int* table, MoveArgs a) {
    const PageBook::PageMove m = a.m[blockIdx.x];
    if (blockIdx.x == 0 && blockIdx.y == 0 && (int)threadIdx.x < a.entries) {
        const PageBook::Entry e = a.e[threadIdx.x];
        table[(size_t)e.row * to_pages + e.block] = e.page;
    }
    const int layer = blockIdx.y / kv_heads, g = blockIdx.y % kv_heads, t = threadIdx.x;
    constexpr size_t BLOCK = 2 * BLOCK_TOKENS * HDP;
    const size_t src = ((size_t)layer * pages + m.src) * kv_heads + g, dst = ((size_t)layer * to_pages + m.dst) * kv_heads + g;
    constexpr int N = BLOCK / 16 / THREADS;
    uint4 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = gload_u4(codes + src * BLOCK + (size_t)(i * THREADS + t) * 16);
#pragma unroll
    for (int i = 0; i < N; ++i) *(uint4*)(to_codes + dst * BLOCK + (size_t)(i * THREADS + t) * 16) = x[i];
    if (t == 0) to_scales[dst] = scales[src];
}

__global__ void clear_kernel(uint4* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
        p[i] = make_uint4(0, 0, 0, 0);
}

}  // namespace
}  // namespace trit

using namespace trit;

struct TritHipPagedCache {
    int device, layers, kv_heads, hd, hdp;
    PageBook book;
    DeviceMemory codes, scales, open, table;
    AttendScratch scratch;
    // The stream of the last call. A call on another one waits for the device
    // first: the books run ahead of it, and a page freed by one call may be
    // the one that the next call writes.
    hipStream_t last = nullptr;
    bool queued = false;
    std::mutex mu;

    TritHipPagedCache(int l, int kvh, int head_dim, int pages, int sequences)
        : device(device_id()), layers(l), kv_heads(kvh), hd(head_dim), hdp(head_dim <= 64 ? 64 : 128),
          book(l, pages, sequences) {}

    size_t block_values() const { return (size_t)2 * BLOCK_TOKENS * hdp; }  // K and V of a head
    void make_pool(int pages, DeviceMemory& c, DeviceMemory& sc, DeviceMemory& tb) const {
        c.alloc((size_t)layers * pages * kv_heads * block_values());
        sc.alloc((size_t)layers * pages * kv_heads * sizeof(float2));
        tb.alloc((size_t)book.sequences() * pages * sizeof(int));
    }
    Pool pool(int layer) const {
        const size_t at = (size_t)layer * book.pages() * kv_heads;
        return Pool{codes.as<uint8_t>() + at * block_values(), scales.as<float2>() + at,
                    open.as<_Float16>() + (size_t)layer * book.sequences() * kv_heads * block_values(), table.as<int>(),
                    book.pages(), kv_heads, hd};
    }
    // Checks that the call can be queued on `stream_`, and in what order.
    hipStream_t enter(void* stream_) {
        int now = -1;
        TRIT_HIP(hipGetDevice(&now));
        if (now != device || (!stream_ && device_id() != device))
            fail("paged cache: it lives on device " + std::to_string(device) + ", the calling thread uses device " +
                 std::to_string(now != device ? now : device_id()));
        hipStream_t s = stream_ ? (hipStream_t)stream_ : stream();
        // An error that an earlier call returned (a failed allocation) is not this call's.
        (void)hipGetLastError();
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        TRIT_HIP(hipStreamIsCapturing(s, &status));
        if (status != hipStreamCaptureStatusNone)
            fail("paged cache: its calls cannot be captured into a graph (their launches hold the sequences' places "
                 "and lengths)");
        if (queued && last != s) TRIT_HIP(hipDeviceSynchronize());
        last = s;
        queued = true;
        return s;
    }

    void write_entries(const std::vector<PageBook::Entry>& entries, hipStream_t s) {
        for (size_t at = 0; at < entries.size(); at += CALL_ENTRIES) {
            TableArgs a;
            const int n = (int)std::min<size_t>(CALL_ENTRIES, entries.size() - at);
            std::copy_n(entries.begin() + (ptrdiff_t)at, n, a.e);
            hipLaunchKernelGGL(table_kernel, dim3(1), dim3(CALL_ENTRIES), 0, s, table.as<int>(), book.pages(), a, n);
            TRIT_HIP(hipGetLastError());
        }
    }
    void copy_rows(const std::vector<PageBook::RowCopy>& rows, TritHipPagedCache& to, hipStream_t s) {
        for (size_t at = 0; at < rows.size(); at += CALL_ENTRIES) {
            CopyArgs a;
            const int n = (int)std::min<size_t>(CALL_ENTRIES, rows.size() - at);
            std::copy_n(rows.begin() + (ptrdiff_t)at, n, a.c);
            const dim3 grid((unsigned)n, (unsigned)(layers * kv_heads), 4);
            auto kernel = hdp == 64 ? row_kernel<64> : row_kernel<128>;
            hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, s, (const _Float16*)open.ptr, book.sequences(),
                               to.open.as<_Float16>(), to.book.sequences(), kv_heads, to.table.as<int>(),
                               to.book.pages(), a);
            TRIT_HIP(hipGetLastError());
        }
    }
    // Moves to `to`, and what changes in its table.
    void move_pages(const std::vector<PageBook::PageMove>& moves, const std::vector<PageBook::Entry>& entries,
                    TritHipPagedCache& to, hipStream_t s) {
        size_t written = 0;
        for (size_t at = 0; at < moves.size(); at += CALL_MOVES) {
            MoveArgs a;
            const int n = (int)std::min<size_t>(CALL_MOVES, moves.size() - at);
            std::copy_n(moves.begin() + (ptrdiff_t)at, n, a.m);
            a.entries = (int)std::min<size_t>(CALL_MOVES, entries.size() - written);
            std::copy_n(entries.begin() + (ptrdiff_t)written, a.entries, a.e);
            written += (size_t)a.entries;
            const dim3 grid((unsigned)n, (unsigned)(layers * kv_heads));
            auto kernel = hdp == 64 ? page_kernel<64> : page_kernel<128>;
            hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, s, (const uint8_t*)codes.ptr, (const float2*)scales.ptr,
                               book.pages(), to.codes.as<uint8_t>(), to.scales.as<float2>(), to.book.pages(), kv_heads,
                               to.table.as<int>(), a);
            TRIT_HIP(hipGetLastError());
        }
        // Pages that several sequences share have more entries than moves.
        to.write_entries({entries.begin() + (ptrdiff_t)written, entries.end()}, s);
    }
};

namespace trit {
namespace {

// Device buffers of the host-memory calls.
struct HostRows {
    DeviceMemory k, v;
    size_t bytes;
    explicit HostRows(long long rows, size_t width) : bytes((size_t)rows * width * 4) {
        k.alloc(bytes);
        v.alloc(bytes);
    }
};

void check_sequences(const char* what, const void* sequences, const void* counts, int n) {
    if (n < 0) fail(std::string(what) + ": a negative number of sequences");
    if (n && (!sequences || !counts)) fail(std::string(what) + ": sequences or rows is NULL");
}

// Whether 4 dims of any row and head are 16 bytes at a 16-byte address.
bool vectors(int hd, const void* k, int64_t ks, const void* v, int64_t vs) {
    return hd % 4 == 0 && ks % 4 == 0 && vs % 4 == 0 && ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
}

// The sum of n row counts, each 0 or more.
long long total_rows(const char* what, const int32_t* rows, int n) {
    long long total = 0;
    for (int i = 0; i < n; ++i) {
        if (rows[i] < 0) fail(std::string(what) + ": a negative number of rows");
        total += rows[i];
    }
    if (total > (1 << 30)) fail(std::string(what) + ": more than 2^30 rows");
    return total;
}

}  // namespace
}  // namespace trit

extern "C" {

int trit_hip_paged_new(int layers, int kv_heads, int head_dim, int pages, int sequences, TritHipPagedCache** out) {
    return guard(-1, [&] {
        if (!out) fail("paged cache: out is NULL");
        if (layers <= 0 || kv_heads <= 0 || pages <= 0 || sequences <= 0)
            fail("paged cache: layers, kv_heads, pages and sequences must be positive");
        if (head_dim <= 0 || head_dim > 128) fail("paged cache: head_dim must be 1 to 128");
        if ((long long)layers * kv_heads > 65535) fail("paged cache: more than 65535 heads in all layers");
        if (pages > (1 << 24) || sequences > 65536) fail("paged cache: more than 2^24 pages or 65536 sequences");
        auto c = std::make_unique<TritHipPagedCache>(layers, kv_heads, head_dim, pages, sequences);
        c->make_pool(pages, c->codes, c->scales, c->table);
        c->open.alloc((size_t)layers * sequences * kv_heads * c->block_values() * 2);
        // Zeros past head_dim, which no append writes.
        hipLaunchKernelGGL(clear_kernel, dim3(1024), dim3(THREADS), 0, c->enter(nullptr), c->open.as<uint4>(),
                           c->open.bytes / 16);
        TRIT_HIP(hipGetLastError());
        c->scratch.make(c->hdp, c->last);
        *out = c.release();
        return 0;
    });
}

void trit_hip_paged_free(TritHipPagedCache* cache) { delete cache; }

int trit_hip_paged_open(TritHipPagedCache* cache, int n, int32_t* out) {
    return guard(-1, [&] {
        if (!cache || (n > 0 && !out)) fail("paged open: cache or out is NULL");
        std::lock_guard<std::mutex> lock(cache->mu);
        cache->book.open(n, out);
        return 0;
    });
}

int trit_hip_paged_fork(TritHipPagedCache* cache, const int32_t* sequences, int n, int32_t* out, void* stream_) {
    return guard(-1, [&] {
        if (!cache || (n > 0 && (!sequences || !out))) fail("paged fork: cache, sequences or out is NULL");
        std::lock_guard<std::mutex> lock(cache->mu);
        const hipStream_t s = cache->enter(stream_);
        cache->copy_rows(cache->book.fork(sequences, n, out), *cache, s);
        return 0;
    });
}

int trit_hip_paged_reorder(TritHipPagedCache* cache, const int32_t* sequences, const int32_t* parents, int n,
                           void* stream_) {
    return guard(-1, [&] {
        if (!cache || (n > 0 && (!sequences || !parents))) fail("paged reorder: cache, sequences or parents is NULL");
        std::lock_guard<std::mutex> lock(cache->mu);
        const hipStream_t s = cache->enter(stream_);
        cache->copy_rows(cache->book.reorder(sequences, parents, n), *cache, s);
        return 0;
    });
}

int trit_hip_paged_copy(TritHipPagedCache* cache, const int32_t* sequences, int n, TritHipPagedCache* into,
                        int32_t* out, void* stream_) {
    return guard(-1, [&] {
        if (!cache || (n > 0 && (!sequences || !out))) fail("paged copy: cache, sequences or out is NULL");
        if (!into) into = cache;
        if (into->layers != cache->layers || into->kv_heads != cache->kv_heads || into->hd != cache->hd)
            fail("paged copy: the caches differ in layers, kv_heads or head_dim");
        std::unique_lock<std::mutex> a(cache->mu, std::defer_lock), b(into->mu, std::defer_lock);
        if (into == cache)
            a.lock();
        else
            std::lock(a, b);
        const hipStream_t s = cache->enter(stream_);
        if (into != cache) into->enter(stream_);
        std::vector<PageBook::RowCopy> rows;
        std::vector<PageBook::PageMove> pages;
        std::vector<PageBook::Entry> entries;
        cache->book.copy(sequences, n, into->book, out, rows, pages, entries);
        cache->move_pages(pages, entries, *into, s);
        cache->copy_rows(rows, *into, s);
        return 0;
    });
}

int trit_hip_paged_close(TritHipPagedCache* cache, const int32_t* sequences, int n) {
    return guard(-1, [&] {
        if (!cache || n < 0 || (n > 0 && !sequences)) fail("paged close: cache or sequences is NULL, or n is negative");
        std::lock_guard<std::mutex> lock(cache->mu);
        cache->book.close(sequences, n);
        return 0;
    });
}

int trit_hip_paged_compact(TritHipPagedCache* cache, void* stream_) {
    return guard(-1, [&] {
        if (!cache) fail("paged compact: cache is NULL");
        std::lock_guard<std::mutex> lock(cache->mu);
        const hipStream_t s = cache->enter(stream_);
        std::vector<PageBook::PageMove> moves;
        std::vector<PageBook::Entry> entries;
        cache->book.compact(moves, entries);
        cache->move_pages(moves, entries, *cache, s);
        return cache->book.pages_in_use();
    });
}

int trit_hip_paged_resize(TritHipPagedCache* cache, int pages, void* stream_) {
    return guard(-1, [&] {
        if (!cache) fail("paged resize: cache is NULL");
        if (pages <= 0 || pages > (1 << 24)) fail("paged resize: 1 to 2^24 pages");
        std::lock_guard<std::mutex> lock(cache->mu);
        PageBook& book = cache->book;
        const int used = book.pages_in_use();
        if (used > pages) fail("paged resize: " + std::to_string(used) + " pages are in use");
        const hipStream_t s = cache->enter(stream_);
        DeviceMemory codes, scales, table;
        cache->make_pool(pages, codes, scales, table);
        std::vector<PageBook::PageMove> moves;
        std::vector<PageBook::Entry> entries;
        book.compact(moves, entries);
        cache->move_pages(moves, {}, *cache, s);
        const size_t page = (size_t)cache->kv_heads * cache->block_values(), scale = (size_t)cache->kv_heads * sizeof(float2);
        for (size_t l = 0; used && l < (size_t)cache->layers; ++l) {
            TRIT_HIP(hipMemcpyAsync(codes.as<uint8_t>() + l * pages * page,
                                    cache->codes.as<uint8_t>() + l * book.pages() * page, used * page,
                                    hipMemcpyDeviceToDevice, s));
            TRIT_HIP(hipMemcpyAsync(scales.as<uint8_t>() + l * pages * scale,
                                    cache->scales.as<uint8_t>() + l * book.pages() * scale, used * scale,
                                    hipMemcpyDeviceToDevice, s));
        }
        // The old arrays are freed below.
        TRIT_HIP(hipStreamSynchronize(s));
        std::swap(cache->codes.ptr, codes.ptr);
        std::swap(cache->codes.bytes, codes.bytes);
        std::swap(cache->scales.ptr, scales.ptr);
        std::swap(cache->scales.bytes, scales.bytes);
        std::swap(cache->table.ptr, table.ptr);
        std::swap(cache->table.bytes, table.bytes);
        book.resize(pages);
        cache->write_entries(book.entries(), s);
        return 0;
    });
}

int trit_hip_paged_length(TritHipPagedCache* cache, int sequence, int layer) {
    return guard(-1, [&] {
        if (!cache) fail("paged length: cache is NULL");
        std::lock_guard<std::mutex> lock(cache->mu);
        return cache->book.length(sequence, layer);
    });
}

int trit_hip_paged_info(TritHipPagedCache* cache, int* pages, int* pages_in_use, int64_t* bytes) {
    return guard(-1, [&] {
        if (!cache) fail("paged info: cache is NULL");
        std::lock_guard<std::mutex> lock(cache->mu);
        if (pages) *pages = cache->book.pages();
        if (pages_in_use) *pages_in_use = cache->book.pages_in_use();
        if (bytes)
            *bytes = (int64_t)(cache->codes.bytes + cache->scales.bytes + cache->open.bytes + cache->table.bytes);
        return 0;
    });
}

int trit_hip_paged_append_device(TritHipPagedCache* cache, int layer, const int32_t* sequences, const int32_t* rows,
                                 int n, const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                                 void* stream_) {
    return guard(-1, [&] {
        if (!cache) fail("paged append: cache is NULL");
        check_sequences("paged append", sequences, rows, n);
        const long long total = total_rows("paged append", rows, n);
        const int64_t width = (int64_t)cache->kv_heads * cache->hd;
        if (total && (!k || !v)) fail("paged append: k or v is NULL");
        if (k_stride < width || v_stride < width) fail("paged append: a row stride is shorter than its heads");
        std::lock_guard<std::mutex> lock(cache->mu);
        const hipStream_t s = cache->enter(stream_);
        std::vector<RowsSeq> seqs;
        int first = 0;
        for (int i = 0; i < n; ++i) {
            seqs.push_back({cache->book.row(sequences[i]), cache->book.length(sequences[i], layer), 0, rows[i], first});
            first += rows[i];
        }
        cache->write_entries(cache->book.append(layer, sequences, rows, n), s);
        for (int at = 0; at < n; at += CALL_SEQS) {
            RowsArgs a;
            const int m = std::min(CALL_SEQS, n - at);
            int most = 0;
            for (int i = 0; i < m; ++i) {
                a.s[i] = seqs[(size_t)(at + i)];
                if (a.s[i].count)
                    most = std::max(most, (a.s[i].len % BLOCK_TOKENS + a.s[i].count + BLOCK_TOKENS - 1) / BLOCK_TOKENS);
            }
            if (!most) continue;
            auto kernel = cache->hdp == 64 ? append_kernel<64> : append_kernel<128>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)most, (unsigned)cache->kv_heads, (unsigned)(2 * m)), dim3(THREADS),
                               0, s, cache->pool(layer), a, k, (long long)k_stride, v, (long long)v_stride,
                               vectors(cache->hd, k, k_stride, v, v_stride));
            TRIT_HIP(hipGetLastError());
        }
        return 0;
    });
}

int trit_hip_paged_append(TritHipPagedCache* cache, int layer, const int32_t* sequences, const int32_t* rows, int n,
                          const float* k, const float* v) {
    return guard(-1, [&] {
        if (!cache) fail("paged append: cache is NULL");
        check_sequences("paged append", sequences, rows, n);
        const long long total = total_rows("paged append", rows, n);
        if (total && (!k || !v)) fail("paged append: k or v is NULL");
        const int64_t width = (int64_t)cache->kv_heads * cache->hd;
        HostRows d(total, (size_t)width);
        const hipStream_t s = stream();
        if (total) {
            TRIT_HIP(hipMemcpyAsync(d.k.ptr, k, d.bytes, hipMemcpyHostToDevice, s));
            TRIT_HIP(hipMemcpyAsync(d.v.ptr, v, d.bytes, hipMemcpyHostToDevice, s));
        }
        if (trit_hip_paged_append_device(cache, layer, sequences, rows, n, d.k.as<float>(), width, d.v.as<float>(),
                                         width, s) != 0)
            fail(std::string(error_text()));
        TRIT_HIP(hipStreamSynchronize(s));
        return 0;
    });
}

int trit_hip_paged_read_device(TritHipPagedCache* cache, int layer, const int32_t* sequences, const int32_t* first,
                               const int32_t* rows, int n, float* k, int64_t k_stride, float* v, int64_t v_stride,
                               void* stream_) {
    return guard(-1, [&] {
        if (!cache) fail("paged read: cache is NULL");
        check_sequences("paged read", sequences, rows, n);
        if (n && !first) fail("paged read: first is NULL");
        const long long total = total_rows("paged read", rows, n);
        const int64_t width = (int64_t)cache->kv_heads * cache->hd;
        if (total && (!k || !v)) fail("paged read: k or v is NULL");
        if (k_stride < width || v_stride < width) fail("paged read: a row stride is shorter than its heads");
        std::lock_guard<std::mutex> lock(cache->mu);
        std::vector<RowsSeq> seqs;
        int at_row = 0;
        for (int i = 0; i < n; ++i) {
            const int len = cache->book.length(sequences[i], layer);
            if (first[i] < 0 || (long long)first[i] + rows[i] > len)
                fail("paged read: rows " + std::to_string(first[i]) + " to " +
                     std::to_string((long long)first[i] + rows[i]) + " of sequence " + std::to_string(sequences[i]) +
                     ", which holds " + std::to_string(len));
            seqs.push_back({cache->book.row(sequences[i]), len, first[i], rows[i], at_row});
            at_row += rows[i];
        }
        const hipStream_t s = cache->enter(stream_);
        for (int at = 0; at < n; at += CALL_SEQS) {
            RowsArgs a;
            const int m = std::min(CALL_SEQS, n - at);
            int most = 0;
            for (int i = 0; i < m; ++i) {
                a.s[i] = seqs[(size_t)(at + i)];
                if (a.s[i].count)
                    most = std::max(most, (a.s[i].at % BLOCK_TOKENS + a.s[i].count + BLOCK_TOKENS - 1) / BLOCK_TOKENS);
            }
            if (!most) continue;
            auto kernel = cache->hdp == 64 ? read_kernel<64> : read_kernel<128>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)most, (unsigned)cache->kv_heads, (unsigned)(2 * m)), dim3(THREADS),
                               0, s, cache->pool(layer), a, k, (long long)k_stride, v, (long long)v_stride,
                               vectors(cache->hd, k, k_stride, v, v_stride));
            TRIT_HIP(hipGetLastError());
        }
        return 0;
    });
}

int trit_hip_paged_read(TritHipPagedCache* cache, int layer, const int32_t* sequences, const int32_t* first,
                        const int32_t* rows, int n, float* k, float* v) {
    return guard(-1, [&] {
        if (!cache) fail("paged read: cache is NULL");
        check_sequences("paged read", sequences, rows, n);
        const long long total = total_rows("paged read", rows, n);
        if (total && (!k || !v)) fail("paged read: k or v is NULL");
        const int64_t width = (int64_t)cache->kv_heads * cache->hd;
        HostRows d(total, (size_t)width);
        const hipStream_t s = stream();
        if (trit_hip_paged_read_device(cache, layer, sequences, first, rows, n, d.k.as<float>(), width, d.v.as<float>(),
                                       width, s) != 0)
            fail(std::string(error_text()));
        if (total) {
            TRIT_HIP(hipMemcpyAsync(k, d.k.ptr, d.bytes, hipMemcpyDeviceToHost, s));
            TRIT_HIP(hipMemcpyAsync(v, d.v.ptr, d.bytes, hipMemcpyDeviceToHost, s));
        }
        TRIT_HIP(hipStreamSynchronize(s));
        return 0;
    });
}

int trit_hip_paged_attention_device(TritHipPagedCache* cache, int layer, const int32_t* sequences,
                                    const int32_t* rows, int n, const float* q, int64_t q_stride, int heads,
                                    float scale, float* out, void* stream_) {
    return guard(-1, [&] {
        if (!cache) fail("paged attention: cache is NULL");
        check_sequences("paged attention", sequences, rows, n);
        const long long total = total_rows("paged attention", rows, n);
        if (total && (!q || !out)) fail("paged attention: q or out is NULL");
        if (heads <= 0 || heads % cache->kv_heads)
            fail("paged attention: the query heads do not share the key heads evenly");
        if (q_stride < (int64_t)heads * cache->hd) fail("paged attention: the query stride is shorter than its heads");
        if (!(scale >= 0.0f && scale < INFINITY)) fail("paged attention: the scale must be 0 (1/sqrt(head_dim)) or more");
        std::lock_guard<std::mutex> lock(cache->mu);
        std::vector<AttendSeq> seqs;
        int first = 0;
        for (int i = 0; i < n; ++i) {
            const int len = cache->book.length(sequences[i], layer);
            if (rows[i] > len)
                fail("paged attention: " + std::to_string(rows[i]) + " query rows of sequence " +
                     std::to_string(sequences[i]) + ", which holds " + std::to_string(len) + " tokens");
            seqs.push_back({cache->book.row(sequences[i]), len, rows[i], first, 0, 0, 0, 0});
            first += rows[i];
        }
        const hipStream_t s = cache->enter(stream_);
        const Pool p = cache->pool(layer);
        AttendArgs a;
        a.q = q;
        a.qs = q_stride;
        a.out = out;
        a.scale = scale != 0.0f ? scale : 1.0f / __builtin_sqrtf((float)cache->hd);
        a.kv_heads = cache->kv_heads;
        a.group = heads / cache->kv_heads;
        a.hd = cache->hd;
        a.codes = p.codes;
        a.scales = p.scales;
        a.table = p.table;
        a.table_stride = p.pages;
        a.f16 = p.open;
        attend(a, seqs, true, cache->scratch, s);
        return 0;
    });
}

int trit_hip_paged_attention(TritHipPagedCache* cache, int layer, const int32_t* sequences, const int32_t* rows, int n,
                             const float* q, int heads, float scale, float* out) {
    return guard(-1, [&] {
        if (!cache) fail("paged attention: cache is NULL");
        check_sequences("paged attention", sequences, rows, n);
        const long long total = total_rows("paged attention", rows, n);
        if (total && (!q || !out)) fail("paged attention: q or out is NULL");
        if (heads <= 0 || heads % cache->kv_heads)
            fail("paged attention: the query heads do not share the key heads evenly");
        HostRows d(total, (size_t)heads * cache->hd);  // k: the queries, v: the output
        const hipStream_t s = stream();
        if (total) TRIT_HIP(hipMemcpyAsync(d.k.ptr, q, d.bytes, hipMemcpyHostToDevice, s));
        if (trit_hip_paged_attention_device(cache, layer, sequences, rows, n, d.k.as<float>(),
                                            (int64_t)heads * cache->hd, heads, scale, d.v.as<float>(), s) != 0)
            fail(std::string(error_text()));
        if (total) TRIT_HIP(hipMemcpyAsync(out, d.v.ptr, d.bytes, hipMemcpyDeviceToHost, s));
        TRIT_HIP(hipStreamSynchronize(s));
        return 0;
    });
}

}  // extern "C"
