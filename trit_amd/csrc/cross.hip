// Cross attention (include/trit_hip.h): the keys and values of encoder states,
// held as f16 in the attention kernel's operand order, and the attention of
// decoder rows to them.
#include <algorithm>
#include <mutex>

#include "../../include/trit_hip.h"
#include "attend.h"
#include "blocks.h"
#include "device.h"
#include "internal.h"

namespace trit {
namespace {

constexpr int THREADS = BLOCK_THREADS;

struct SetSeq {
    int slot, keys;
    int first;  // its first row in the caller's arrays
};
struct SetArgs {
    SetSeq s[CALL_SEQS];
};

// Workgroup (x, g, 2 i + which): block x of keys (which 0) or values (1) of
// head g of the i-th slot, zero past its keys and past head_dim. (Values of
// keys that are not there meet probabilities of 0.)
template <int HDP, bool V>
__device__ __forceinline__ void set_block(_Float16* to, int hd, int keys, const float* rows, long long stride,
                                          bool aligned, _Float16* out) {
    constexpr int G = BlockShare<HDP>::GROUPS;
    const int t = threadIdx.x, first = blockIdx.x * BLOCK_TOKENS;
    float h[4 * G];
    load_share<HDP, V>(rows, stride, first, keys, hd, aligned, h);
#pragma unroll
    for (int i = 0; i < G; ++i) {
        int tok, e;
        share_at<HDP, V>(i, tok, e);
        _Float16 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool valid = first + tok + (V ? j : 0) < keys && e + (V ? 0 : j) < hd;
            x[j] = valid ? held(h[4 * i + j]) : (_Float16)0.0f;
        }
        __builtin_memcpy(out + half_at<HDP, V>(tok, e), x, 8);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BLOCK_TOKENS * HDP / 8; i += THREADS) *(uint4*)(to + (i + t) * 8) = *(const uint4*)(out + (i + t) * 8);
}
template <int HDP>
__global__ __launch_bounds__(THREADS) void set_kernel(_Float16* states, int blocks, int kv_heads, int hd, SetArgs a,
                                                      const float* k, long long ks, const float* v, long long vs,
                                                      bool aligned) {
    __shared__ __align__(16) _Float16 out[BLOCK_TOKENS * HDP];
    const int g = blockIdx.y;
    const SetSeq s = a.s[blockIdx.z / 2];
    if ((int)blockIdx.x * BLOCK_TOKENS >= s.keys) return;
    _Float16* to =
        states + (((size_t)s.slot * kv_heads + g) * blocks + blockIdx.x) * 2 * (BLOCK_TOKENS * HDP);
    if (blockIdx.z % 2)
        set_block<HDP, true>(to + BLOCK_TOKENS * HDP, hd, s.keys, v + (size_t)s.first * vs + (size_t)g * hd, vs, aligned, out);
    else
        set_block<HDP, false>(to, hd, s.keys, k + (size_t)s.first * ks + (size_t)g * hd, ks, aligned, out);
}

}  // namespace
}  // namespace trit

using namespace trit;

struct TritHipCross {
    int device, layers, kv_heads, hd, hdp, slots, max_keys, blocks;
    DeviceMemory states;
    AttendScratch scratch;
    std::vector<int> keys;  // by layer and slot; -1: never set
    // The stream of the last call; one on another waits for the device first.
    hipStream_t last = nullptr;
    bool queued = false;
    std::mutex mu;

    size_t layer_values() const { return (size_t)slots * kv_heads * blocks * 2 * BLOCK_TOKENS * hdp; }

    // Checks that the call can be queued on `stream_`, and in what order.
    hipStream_t enter(void* stream_) {
        int now = -1;
        TRIT_HIP(hipGetDevice(&now));
        if (now != device || (!stream_ && device_id() != device))
            fail("cross attention: the states live on device " + std::to_string(device) +
                 ", the calling thread uses device " + std::to_string(now != device ? now : device_id()));
        hipStream_t s = stream_ ? (hipStream_t)stream_ : stream();
        // An error that an earlier call returned (a failed allocation) is not this call's.
        (void)hipGetLastError();
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        TRIT_HIP(hipStreamIsCapturing(s, &status));
        if (status != hipStreamCaptureStatusNone)
            fail("cross attention: its calls cannot be captured into a graph (their launches hold the states' "
                 "lengths)");
        if (queued && last != s) TRIT_HIP(hipDeviceSynchronize());
        last = s;
        queued = true;
        return s;
    }
};

namespace trit {
namespace {

void check_slots(const TritHipCross& c, const char* what, int layer, const int32_t* slots, int n) {
    if (layer < 0 || layer >= c.layers)
        fail(std::string(what) + ": layer " + std::to_string(layer) + " of " + std::to_string(c.layers));
    for (int i = 0; i < n; ++i)
        if (slots[i] < 0 || slots[i] >= c.slots)
            fail(std::string(what) + ": slot " + std::to_string(slots[i]) + " of " + std::to_string(c.slots));
}

long long sum_rows(const char* what, const int32_t* slots, const int32_t* rows, int n) {
    if (n < 0) fail(std::string(what) + ": a negative number of slots");
    if (n && (!slots || !rows)) fail(std::string(what) + ": slots or counts is NULL");
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

int trit_hip_cross_new(int layers, int kv_heads, int head_dim, int slots, int max_keys, TritHipCross** out) {
    return guard(-1, [&] {
        if (!out) fail("cross attention: out is NULL");
        if (layers <= 0 || kv_heads <= 0 || slots <= 0 || max_keys <= 0)
            fail("cross attention: layers, kv_heads, slots and max_keys must be positive");
        if (head_dim <= 0 || head_dim > 128) fail("cross attention: head_dim must be 1 to 128");
        if (kv_heads > 65535 || slots > (1 << 20) || layers > (1 << 16) || max_keys > (1 << 26))
            fail("cross attention: at most 65535 heads, 2^20 slots, 2^16 layers and 2^26 keys");
        // (Within those the number of bytes may pass 64 bits.)
        const int wide = head_dim <= 64 ? 64 : 128, most = (max_keys + BLOCK_TOKENS - 1) / BLOCK_TOKENS;
        if ((double)layers * slots * kv_heads * most * (BLOCK_TOKENS * wide * 4.0) > 0x1p48)
            fail("cross attention: states of more memory than a device holds");
        auto c = std::make_unique<TritHipCross>();
        c->device = device_id();
        c->layers = layers;
        c->kv_heads = kv_heads;
        c->hd = head_dim;
        c->hdp = wide;
        c->slots = slots;
        c->max_keys = max_keys;
        c->blocks = most;
        c->states.alloc((size_t)layers * c->layer_values() * 2);
        c->keys.assign((size_t)layers * slots, -1);
        c->scratch.make(c->hdp, c->enter(nullptr));
        *out = c.release();
        return 0;
    });
}

void trit_hip_cross_free(TritHipCross* cross) { delete cross; }

int trit_hip_cross_keys(TritHipCross* cross, int layer, int slot) {
    return guard(-1, [&] {
        if (!cross) fail("cross keys: cross is NULL");
        check_slots(*cross, "cross keys", layer, &slot, 1);
        std::lock_guard<std::mutex> lock(cross->mu);
        const int keys = cross->keys[(size_t)layer * cross->slots + slot];
        if (keys < 0) fail("cross keys: slot " + std::to_string(slot) + " was never set");
        return keys;
    });
}

int trit_hip_cross_set_device(TritHipCross* cross, int layer, const int32_t* slots, const int32_t* keys, int n,
                              const float* k, int64_t k_stride, const float* v, int64_t v_stride, void* stream_) {
    return guard(-1, [&] {
        if (!cross) fail("cross set: cross is NULL");
        const long long total = sum_rows("cross set", slots, keys, n);
        check_slots(*cross, "cross set", layer, slots, n);
        const int64_t width = (int64_t)cross->kv_heads * cross->hd;
        if (total && (!k || !v)) fail("cross set: k or v is NULL");
        if (k_stride < width || v_stride < width) fail("cross set: a row stride is shorter than its heads");
        std::vector<int> named(slots, slots + n);
        std::sort(named.begin(), named.end());
        if (std::adjacent_find(named.begin(), named.end()) != named.end()) fail("cross set: a slot is named twice");
        for (int i = 0; i < n; ++i)
            if (keys[i] > cross->max_keys)
                fail("cross set: " + std::to_string(keys[i]) + " keys where a slot holds " +
                     std::to_string(cross->max_keys));
        std::lock_guard<std::mutex> lock(cross->mu);
        const hipStream_t s = cross->enter(stream_);
        int first = 0;
        for (int at = 0; at < n; at += CALL_SEQS) {
            SetArgs a;
            const int m = std::min(CALL_SEQS, n - at);
            int most = 0;
            for (int i = 0; i < m; ++i) {
                a.s[i] = {slots[at + i], keys[at + i], first};
                first += keys[at + i];
                most = std::max(most, (keys[at + i] + BLOCK_TOKENS - 1) / BLOCK_TOKENS);
                cross->keys[(size_t)layer * cross->slots + slots[at + i]] = keys[at + i];
            }
            if (!most) continue;
            auto kernel = cross->hdp == 64 ? set_kernel<64> : set_kernel<128>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)most, (unsigned)cross->kv_heads, (unsigned)(2 * m)), dim3(THREADS),
                               0, s, cross->states.as<_Float16>() + (size_t)layer * cross->layer_values(), cross->blocks,
                               cross->kv_heads, cross->hd, a, k, (long long)k_stride, v, (long long)v_stride,
                               cross->hd % 4 == 0 && k_stride % 4 == 0 && v_stride % 4 == 0 &&
                                   ((uintptr_t)k | (uintptr_t)v) % 16 == 0);
            TRIT_HIP(hipGetLastError());
        }
        return 0;
    });
}

int trit_hip_cross_set(TritHipCross* cross, int layer, const int32_t* slots, const int32_t* keys, int n, const float* k,
                       const float* v) {
    return guard(-1, [&] {
        if (!cross) fail("cross set: cross is NULL");
        const long long total = sum_rows("cross set", slots, keys, n);
        if (total && (!k || !v)) fail("cross set: k or v is NULL");
        const int64_t width = (int64_t)cross->kv_heads * cross->hd;
        const size_t bytes = (size_t)total * width * 4;
        DeviceMemory dk(bytes), dv(bytes);
        const hipStream_t s = stream();
        if (total) {
            TRIT_HIP(hipMemcpyAsync(dk.ptr, k, bytes, hipMemcpyHostToDevice, s));
            TRIT_HIP(hipMemcpyAsync(dv.ptr, v, bytes, hipMemcpyHostToDevice, s));
        }
        if (trit_hip_cross_set_device(cross, layer, slots, keys, n, dk.as<float>(), width, dv.as<float>(), width, s) != 0)
            fail(std::string(error_text()));
        TRIT_HIP(hipStreamSynchronize(s));
        return 0;
    });
}

int trit_hip_cross_attention_device(TritHipCross* cross, int layer, const int32_t* slots, const int32_t* rows, int n,
                                    const float* q, int64_t q_stride, int heads, float scale, float* out,
                                    void* stream_) {
    return guard(-1, [&] {
        if (!cross) fail("cross attention: cross is NULL");
        const long long total = sum_rows("cross attention", slots, rows, n);
        check_slots(*cross, "cross attention", layer, slots, n);
        if (total && (!q || !out)) fail("cross attention: q or out is NULL");
        if (heads <= 0 || heads % cross->kv_heads)
            fail("cross attention: the query heads do not share the key heads evenly");
        if (q_stride < (int64_t)heads * cross->hd) fail("cross attention: the query stride is shorter than its heads");
        if (!(scale >= 0.0f && scale < INFINITY)) fail("cross attention: the scale must be 0 (1/sqrt(head_dim)) or more");
        std::lock_guard<std::mutex> lock(cross->mu);
        std::vector<AttendSeq> seqs;
        int first = 0;
        for (int i = 0; i < n; ++i) {
            const int keys = cross->keys[(size_t)layer * cross->slots + slots[i]];
            if (keys < 0)
                fail("cross attention: slot " + std::to_string(slots[i]) + " of layer " + std::to_string(layer) +
                     " was never set");
            seqs.push_back({slots[i], keys, rows[i], first, 0, 0, 0, 0});
            first += rows[i];
        }
        const hipStream_t s = cross->enter(stream_);
        AttendArgs a;
        a.q = q;
        a.qs = q_stride;
        a.out = out;
        a.scale = scale != 0.0f ? scale : 1.0f / __builtin_sqrtf((float)cross->hd);
        a.kv_heads = cross->kv_heads;
        a.group = heads / cross->kv_heads;
        a.hd = cross->hd;
        a.f16 = cross->states.as<_Float16>() + (size_t)layer * cross->layer_values();
        a.blocks = cross->blocks;
        attend(a, seqs, false, cross->scratch, s);
        return 0;
    });
}

int trit_hip_cross_attention(TritHipCross* cross, int layer, const int32_t* slots, const int32_t* rows, int n,
                             const float* q, int heads, float scale, float* out) {
    return guard(-1, [&] {
        if (!cross) fail("cross attention: cross is NULL");
        const long long total = sum_rows("cross attention", slots, rows, n);
        if (total && (!q || !out)) fail("cross attention: q or out is NULL");
        if (heads <= 0 || heads % cross->kv_heads)
            fail("cross attention: the query heads do not share the key heads evenly");
        const int64_t width = (int64_t)heads * cross->hd;
        const size_t bytes = (size_t)total * width * 4;
        DeviceMemory dq(bytes), dout(bytes);
        const hipStream_t s = stream();
        if (total) TRIT_HIP(hipMemcpyAsync(dq.ptr, q, bytes, hipMemcpyHostToDevice, s));
        if (trit_hip_cross_attention_device(cross, layer, slots, rows, n, dq.as<float>(), width, heads, scale,
                                            dout.as<float>(), s) != 0)
            fail(std::string(error_text()));
        if (total) TRIT_HIP(hipMemcpyAsync(out, dout.ptr, bytes, hipMemcpyDeviceToHost, s));
        TRIT_HIP(hipStreamSynchronize(s));
        return 0;
    });
}

}  // extern "C"
