// ops_kv4_attention.hip -- lpp_kv4_attention, lpp_kv4_attention_workspace:
// attention of a few new rows over the cache of 4 bits, and the weight each
// position got.
#include "kv4.hpp"

namespace lpp {
namespace {

using namespace dev;

constexpr int kThreads = 256;

__device__ __forceinline__ int rows_end(int start, int row, int seq_len) {
    return static_cast<int>(min(max(static_cast<long long>(start) + row + 1, 0ll), static_cast<long long>(seq_len)));
}

// q . (the row's values), every lane the whole of it.
__device__ __forceinline__ float row_dot(const uint32_t* codes, const uint32_t* scales, const float* q, int head_size) {
    float s = 0.0f;
    for (int w = 0; w < head_size / 8; ++w) {
        const half8_t k = kv4_values(codes[w], scales[w / 4]);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(static_cast<float>(k[e]), q[8 * w + e], s);
    }
    return s;
}

// One wavefront per (sequence, row, query head); a lane has one position's score, then head_size / 64 output values.
// (maximum, sum) of every row and head are left in `stats` for the weights.
__global__ __launch_bounds__(kWave) void attend_kernel(float* __restrict__ out, const float* __restrict__ q, Kv4Layer cache,
                                                       const int* __restrict__ starts, float2* __restrict__ stats, int n_q, int n_heads,
                                                       int n_kv_heads, int head_size, int seq_len, float scale) {
    const int head = blockIdx.x % n_heads, row = blockIdx.x / n_heads, s = blockIdx.y, lane = lane_id();
    const int end = rows_end(starts[s], row, seq_len);
    const size_t at = (static_cast<size_t>(s) * n_q + row) * n_heads + head;
    const float* qv = q + at * head_size;
    const size_t base = (static_cast<size_t>(s) * n_kv_heads + head / (n_heads / n_kv_heads)) * seq_len;
    const int words = head_size / 8, groups = head_size / kKv4Group;
    float top = -INFINITY, sum = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int p0 = 0; p0 < end; p0 += kWave) {
        const int p = p0 + lane;
        const float score = p < end ? scale * row_dot(cache.codes[0] + (base + p) * words, cache.scales[0] + (base + p) * groups, qv, head_size) : -INFINITY;
        const float grown = fmaxf(top, wave_max(score));
        const float weight = expf(score - grown), correction = top == -INFINITY ? 0.0f : expf(top - grown);
        top = grown;
        sum = sum * correction + wave_sum(weight);
        for (int d = 0; d < head_size / kWave; ++d) acc[d] *= correction;
        const int count = min(kWave, end - p0);
        for (int j = 0; j < count; ++j) {
            const float w = __shfl(weight, j);
            for (int d = 0; d < head_size / kWave; ++d) {
                const int e = d * kWave + lane;
                const size_t r = base + p0 + j;
                const half8_t v = kv4_values(cache.codes[1][r * words + e / 8], cache.scales[1][r * groups + e / kKv4Group]);
                acc[d] = fmaf(w, static_cast<float>(v[e % 8]), acc[d]);
            }
        }
    }
    for (int d = 0; d < head_size / kWave; ++d) out[at * head_size + d * kWave + lane] = end > 0 ? acc[d] / sum : 0.0f;
    if (lane == 0) stats[at] = make_float2(top, sum);
}

// One thread per position of a sequence and KV head.
__global__ __launch_bounds__(kThreads) void mass_kernel(float* __restrict__ mass, const float* __restrict__ q, Kv4Layer cache,
                                                        const int* __restrict__ starts, const float2* __restrict__ stats, int n_q, int n_heads,
                                                        int n_kv_heads, int head_size, int seq_len, float scale) {
    const int p = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x), kvh = blockIdx.y, s = blockIdx.z;
    const int shared = n_heads / n_kv_heads;
    if (p >= rows_end(starts[s], n_q - 1, seq_len)) return;
    const size_t at = (static_cast<size_t>(s) * n_kv_heads + kvh) * seq_len + p;
    float total = 0.0f;
    for (int row = 0; row < n_q; ++row) {
        if (p >= rows_end(starts[s], row, seq_len)) continue;
        for (int h = kvh * shared; h < (kvh + 1) * shared; ++h) {
            const size_t r = (static_cast<size_t>(s) * n_q + row) * n_heads + h;
            const float score = scale * row_dot(cache.codes[0] + at * (head_size / 8), cache.scales[0] + at * (head_size / kKv4Group), q + r * head_size, head_size);
            total += expf(score - stats[r].x) / stats[r].y;
        }
    }
    mass[at] += total;
}

lpp_status check(const char* who, const lpp_kv4_shape* shape, int n_heads, int n_q) {
    LPP_TRY(kv4_check_shape(who, shape));
    LPP_REQUIRE(n_heads > 0 && n_heads % shape->n_kv_heads == 0, "%s: n_heads = %d must be a positive multiple of n_kv_heads = %d", who, n_heads,
                shape->n_kv_heads);
    LPP_REQUIRE(n_heads / shape->n_kv_heads <= kMaxSharedHeads, "%s: %d query heads to a KV head are more than %d", who, n_heads / shape->n_kv_heads,
                kMaxSharedHeads);
    LPP_REQUIRE(n_q > 0 && n_q <= shape->seq_len, "%s: n_q = %d, room for %d", who, n_q, shape->seq_len);
    LPP_REQUIRE(static_cast<long long>(n_q) * n_heads <= 0x7fffffffll && shape->n_seqs <= 65535 && shape->n_kv_heads <= 65535,
                "%s: n_q = %d, n_heads = %d, n_seqs = %d", who, n_q, n_heads, shape->n_seqs);
    return LPP_OK;
}

}  // namespace
}  // namespace lpp

extern "C" {

lpp_status lpp_kv4_attention_workspace(const lpp_kv4_shape* shape, int n_heads, int n_q, size_t* bytes) {
    using namespace lpp;
    LPP_TRY(check("lpp_kv4_attention_workspace", shape, n_heads, n_q));
    LPP_REQUIRE(bytes != nullptr, "lpp_kv4_attention_workspace: null output");
    *bytes = static_cast<size_t>(shape->n_seqs) * n_q * n_heads * sizeof(float2);
    return LPP_OK;
}

lpp_status lpp_kv4_attention(float* d_out, const float* d_q, const void* d_cache, const lpp_kv4_shape* shape, int layer, int n_heads, int n_q,
                             const int* d_starts, float* d_mass, void* d_workspace, size_t workspace_bytes) {
    using namespace lpp;
    LPP_TRY(kv4_check_cache("lpp_kv4_attention", d_cache, shape, layer));
    LPP_TRY(check("lpp_kv4_attention", shape, n_heads, n_q));
    LPP_REQUIRE(d_out && d_q && d_starts && d_workspace, "lpp_kv4_attention: null pointer");
    LPP_REQUIRE(reinterpret_cast<uintptr_t>(d_out) % 16 == 0 && reinterpret_cast<uintptr_t>(d_q) % 16 == 0 && reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0,
                "lpp_kv4_attention: d_out, d_q and d_workspace must start at multiples of 16 bytes");
    size_t need = 0;
    LPP_TRY(lpp_kv4_attention_workspace(shape, n_heads, n_q, &need));
    LPP_REQUIRE(workspace_bytes >= need, "lpp_kv4_attention: a workspace of %zu bytes, %zu are needed", workspace_bytes, need);
    const size_t rows_bytes = static_cast<size_t>(shape->n_seqs) * n_q * n_heads * shape->head_size * 4;
    LPP_REQUIRE(!ranges_overlap(d_out, rows_bytes, d_q, rows_bytes), "lpp_kv4_attention: d_out overlaps d_q");
    const Kv4Layer cache = kv4_layer(d_cache, *shape, layer);
    const float scale = 1.0f / sqrtf(static_cast<float>(shape->head_size));
    hipLaunchKernelGGL(attend_kernel, dim3(n_q * n_heads, shape->n_seqs), dim3(kWave), 0, stream(), d_out, d_q, cache, d_starts,
                       static_cast<float2*>(d_workspace), n_q, n_heads, shape->n_kv_heads, shape->head_size, shape->seq_len, scale);
    LPP_CHECK_LAUNCH("attend_kernel");
    if (d_mass != nullptr) {
        hipLaunchKernelGGL(mass_kernel, dim3((shape->seq_len + kThreads - 1) / kThreads, shape->n_kv_heads, shape->n_seqs), dim3(kThreads), 0, stream(),
                           d_mass + kv4_layer_rows(*shape) * layer, d_q, cache, d_starts, static_cast<const float2*>(d_workspace), n_q, n_heads,
                           shape->n_kv_heads, shape->head_size, shape->seq_len, scale);
        LPP_CHECK_LAUNCH("mass_kernel");
    }
    return LPP_OK;
}

}  // extern "C"
