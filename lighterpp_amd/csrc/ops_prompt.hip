// ops_prompt.hip -- lpp_prompt_attention: causal attention of whole prompts,
// packed one behind the other.
#include "kv4.hpp"

namespace lpp {
namespace {

using namespace dev;

// One wavefront per (row, query head); a lane has one position's score, then head_size / 64 output values.
template <typename T>
__global__ __launch_bounds__(kWave) void prompt_kernel(T* __restrict__ out, const T* __restrict__ q, const half_t* __restrict__ k,
                                                       const half_t* __restrict__ v, const int* __restrict__ offsets, int n_seqs,
                                                       int n_heads, int shared, int head_size, int q_stride, int kv_stride, int out_stride, float scale) {
    const int head = blockIdx.x % n_heads, row = blockIdx.x / n_heads, lane = lane_id();
    int first = 0;
    if (offsets != nullptr) {
        const int s = sequence_of_row(offsets + 1, n_seqs, row);
        if (s >= n_seqs) return;
        first = max(offsets[s], 0);
        if (row < first) return;
    }
    const T* qv = q + static_cast<size_t>(row) * q_stride + head * head_size;
    const half_t* kh = k + head / shared * head_size;
    const half_t* vh = v + head / shared * head_size;
    float top = -INFINITY, sum = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int p0 = first; p0 <= row; p0 += kWave) {
        const int p = p0 + lane;
        float score = -INFINITY;
        if (p <= row) {
            score = 0.0f;
            for (int e = 0; e < head_size; ++e) score = fmaf(static_cast<float>(kh[static_cast<size_t>(p) * kv_stride + e]), static_cast<float>(qv[e]), score);
            score *= scale;
        }
        const float grown = fmaxf(top, wave_max(score));
        const float weight = expf(score - grown), correction = top == -INFINITY ? 0.0f : expf(top - grown);
        top = grown;
        sum = sum * correction + wave_sum(weight);
        const int count = min(kWave, row + 1 - p0);
        for (int d = 0; d < head_size / kWave; ++d) {
            acc[d] *= correction;
            for (int j = 0; j < count; ++j)
                acc[d] = fmaf(__shfl(weight, j), static_cast<float>(vh[static_cast<size_t>(p0 + j) * kv_stride + d * kWave + lane]), acc[d]);
        }
    }
    for (int d = 0; d < head_size / kWave; ++d) out[static_cast<size_t>(row) * out_stride + head * head_size + d * kWave + lane] = static_cast<T>(acc[d] / sum);
}

}  // namespace
}  // namespace lpp

extern "C" {

lpp_status lpp_prompt_attention(void* d_out, const void* d_q, const lpp_half* d_k, const lpp_half* d_v, int type, const int* d_offsets, int n_seqs,
                                int n_tokens, int n_heads, int n_kv_heads, int head_size, int q_stride, int kv_stride, int out_stride) {
    using namespace lpp;
    LPP_REQUIRE(type == LPP_F32 || type == LPP_F16, "lpp_prompt_attention: type = %d", type);
    LPP_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0,
                "lpp_prompt_attention: n_heads = %d must be a positive multiple of n_kv_heads = %d", n_heads, n_kv_heads);
    LPP_REQUIRE(n_heads / n_kv_heads <= kMaxSharedHeads, "lpp_prompt_attention: %d query heads to a KV head are more than %d", n_heads / n_kv_heads,
                kMaxSharedHeads);
    LPP_REQUIRE(head_size == 64 || head_size == 128, "lpp_prompt_attention: head_size = %d is neither 64 nor 128", head_size);
    LPP_REQUIRE(n_tokens >= 0 && n_seqs > 0 && (d_offsets != nullptr || n_seqs == 1), "lpp_prompt_attention: n_tokens = %d, n_seqs = %d%s", n_tokens, n_seqs,
                d_offsets ? "" : " without offsets");
    const long long width = static_cast<long long>(n_heads) * head_size, kv_width = static_cast<long long>(n_kv_heads) * head_size;
    LPP_REQUIRE(q_stride >= width && out_stride >= width && kv_stride >= kv_width,
                "lpp_prompt_attention: strides of %d (q), %d (k, v), %d (out) for rows of %lld and %lld", q_stride, kv_stride, out_stride, width, kv_width);
    if (n_tokens == 0) return LPP_OK;
    LPP_REQUIRE(d_out && d_q && d_k && d_v, "lpp_prompt_attention: null pointer");
    const int size = type == LPP_F32 ? 4 : 2, per16 = 16 / size;
    const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    LPP_REQUIRE(aligned(d_out) && aligned(d_q) && aligned(d_k) && aligned(d_v) && q_stride % per16 == 0 && out_stride % per16 == 0 && kv_stride % 8 == 0,
                "lpp_prompt_attention: rows must start at multiples of 16 bytes");
    const auto bytes = [&](int stride, long long row, int of) { return (static_cast<size_t>(n_tokens - 1) * stride + row) * of; };
    const size_t out_bytes = bytes(out_stride, width, size), q_bytes = bytes(q_stride, width, size), kv_bytes = bytes(kv_stride, kv_width, 2);
    LPP_REQUIRE(!ranges_overlap(d_out, out_bytes, d_q, q_bytes) && !ranges_overlap(d_out, out_bytes, d_k, kv_bytes) &&
                    !ranges_overlap(d_out, out_bytes, d_v, kv_bytes),
                "lpp_prompt_attention: d_out overlaps an input");
    const float scale = 1.0f / sqrtf(static_cast<float>(head_size));
    const dim3 grid(static_cast<unsigned>(n_tokens) * n_heads);
    if (type == LPP_F32)
        hipLaunchKernelGGL((prompt_kernel<float>), grid, dim3(dev::kWave), 0, stream(), static_cast<float*>(d_out), static_cast<const float*>(d_q),
                           reinterpret_cast<const dev::half_t*>(d_k), reinterpret_cast<const dev::half_t*>(d_v), d_offsets, n_seqs, n_heads,
                           n_heads / n_kv_heads, head_size, q_stride, kv_stride, out_stride, scale);
    else
        hipLaunchKernelGGL((prompt_kernel<dev::half_t>), grid, dim3(dev::kWave), 0, stream(), static_cast<dev::half_t*>(d_out),
                           static_cast<const dev::half_t*>(d_q), reinterpret_cast<const dev::half_t*>(d_k), reinterpret_cast<const dev::half_t*>(d_v),
                           d_offsets, n_seqs, n_heads, n_heads / n_kv_heads, head_size, q_stride, kv_stride, out_stride, scale);
    LPP_CHECK_LAUNCH("prompt_kernel");
    return LPP_OK;
}

}  // extern "C"
