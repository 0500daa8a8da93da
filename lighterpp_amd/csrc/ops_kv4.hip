// ops_kv4.hip -- lpp_kv4_bytes, lpp_kv4_store, lpp_kv4_load, lpp_kv4_evict: rows
// into and out of the cache of 4 bits, and its reduction by accumulated weight.
#include "kv4.hpp"

namespace lpp {
namespace {

using namespace dev;

constexpr int kStoreThreads = 256;

// The 32 values of a group lie in four adjacent lanes, eight each.
__device__ __forceinline__ float quad_min(float v) {
    v = fminf(v, dpp_move<kDppXor1>(v));
    return fminf(v, dpp_move<kDppXor2>(v));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, dpp_move<kDppXor1>(v));
    return fmaxf(v, dpp_move<kDppXor2>(v));
}
__device__ __forceinline__ int quad_or(int v) {
    v |= dpp_move_i<kDppXor1>(v);
    return v | dpp_move_i<kDppXor2>(v);
}

// The integer nearest to (x - low) / scale, in 0 .. 15.  In fp32 the quotient is off by less than 16 * 3 * 2^-24 where the
// result is not cut, so only a quotient within 1e-5 of a border is formed again, in 64 bits (one value in 50000).
__device__ __forceinline__ uint32_t code_of(float x, float low, float scale, float inverse) {
    const float t = (x - low) * inverse;
    float k = rintf(t);
    if (fabsf(t - k) > 0.5f - 1e-5f && scale > 0.0f)
        k = static_cast<float>(rint((static_cast<double>(x) - static_cast<double>(low)) / static_cast<double>(scale)));
    return static_cast<uint32_t>(fminf(fmaxf(k, 0.0f), 15.0f));
}

// One wavefront per row of K or V; a lane has a word's eight values.
template <typename T>
__global__ __launch_bounds__(kStoreThreads) void store_kernel(Kv4Layer to, const T* __restrict__ k, const T* __restrict__ v, int stride,
                                                              const int* __restrict__ offsets, const int* __restrict__ starts, int n_tokens,
                                                              int n_seqs, int n_kv_heads, int head_size, int seq_len) {
    const int wave = wave_index(), lane = lane_id();
    const int row = static_cast<int>(blockIdx.x) * 2 + wave / 2, which = wave & 1;
    if (row >= n_tokens) return;
    int s, first;
    if (offsets != nullptr) {
        s = sequence_of_row(offsets + 1, n_seqs, row);
        if (s >= n_seqs) return;
        first = max(offsets[s], 0);
        if (row < first) return;
    } else {
        const int each = n_tokens / n_seqs;
        s = row / each;
        first = s * each;
    }
    const long long pos = (starts != nullptr ? static_cast<long long>(starts[s]) : 0ll) + row - first;
    if (pos < 0 || pos >= seq_len) return;
    const T* from = (which ? v : k) + static_cast<size_t>(row) * stride;
    uint32_t* codes = to.codes[which];
    uint32_t* scales = to.scales[which];
    const int words = n_kv_heads * head_size / 8, per_head = head_size / 8;
    for (int w = lane; w < words; w += kWave) {
        float x[8];
        if constexpr (sizeof(T) == 2) {
            const half8_t h = as_half8(load16(from + 8 * w));
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(h[e]);
        } else {
            const floatx4 a = as_float4(load16(from + 8 * w)), b = as_float4(load16(from + 8 * w + 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = a[e];
                x[4 + e] = b[e];
            }
        }
        float least = x[0], most = x[0];
        int bad = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            least = fminf(least, x[e]);
            most = fmaxf(most, x[e]);
            bad |= fabsf(x[e]) <= 32768.0f ? 0 : 1;
        }
        least = quad_min(least);
        most = quad_max(most);
        bad = quad_or(bad);
        // (a row's words are whole groups, so a group's four lanes are all here)
        const half_t low16 = static_cast<half_t>(least), scale16 = static_cast<half_t>((most - least) / 15.0f);
        const float low = static_cast<float>(low16), scale = static_cast<float>(scale16);
        const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
        uint32_t word = 0, pair = 0x7E000000u;
        if (!bad) {
#pragma unroll
            for (int e = 0; e < 8; ++e) word |= code_of(x[e], low, scale, inverse) << (4 * (e / 2) + 16 * (e & 1));
            pair = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, scale16)) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, low16)) << 16;
        }
        const int head = w / per_head, in_head = w - head * per_head;
        const size_t at = (static_cast<size_t>(s) * n_kv_heads + head) * seq_len + static_cast<size_t>(pos);
        codes[at * per_head + in_head] = word;
        if ((w & 3) == 0) scales[at * (per_head / 4) + in_head / 4] = pair;
    }
}

// One thread per word; blockIdx.y: sequences and KV heads, blockIdx.z: K, V.
constexpr int kLoadThreads = 256;
__global__ __launch_bounds__(kLoadThreads) void load_kernel(half_t* __restrict__ k, half_t* __restrict__ v, Kv4Layer from, int planes,
                                                            int per_head, int seq_len, int first, int count) {
    const size_t words = static_cast<size_t>(count) * per_head;
    const size_t i = static_cast<size_t>(blockIdx.x) * kLoadThreads + threadIdx.x;
    if (i >= words) return;
    const Kv4Reader read;
    half_t* to = blockIdx.z ? v : k;
    const uint32_t* codes = from.codes[blockIdx.z];
    const uint32_t* scales = from.scales[blockIdx.z];
    for (int plane = blockIdx.y; plane < planes; plane += gridDim.y) {
        const size_t at = (static_cast<size_t>(plane) * seq_len + first) * per_head + i;
        const half8_t values = read(codes[at], scales[at / 4]);
        *reinterpret_cast<half8_t*>(to + (static_cast<size_t>(plane) * words + i) * 8) = values;
    }
}

// ---------------------------------------------------------------------------
// Reduction by accumulated weight
// ---------------------------------------------------------------------------

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;

// Weights as integers in the same order: NaN above everything, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float mass) {
    if (mass != mass) return 0xffffffffu;
    const uint32_t bits = __float_as_uint(mass + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// One workgroup per sequence and KV head: the keep - recent positions of largest weight among the first n - recent, by the bits of the
// smallest one kept, eight at a time from the top (256 counts a pass), then the list in order.
__global__ __launch_bounds__(kSelectThreads) void select_kernel(int* __restrict__ kept, int* __restrict__ dst_lengths, const float* __restrict__ mass,
                                                                const int* __restrict__ lengths, int n_kv_heads, int seq_len, int keep, int recent) {
    __shared__ int counts[256];
    __shared__ int wave_counts[2][kSelectWaves];
    __shared__ int found_bin, found_above;
    const int plane = blockIdx.x, s = plane / n_kv_heads, lane = lane_id(), wave = wave_index();
    const int n = min(max(lengths[s], 0), seq_len), most = min(n, keep);
    int* list = kept + static_cast<size_t>(plane) * keep;
    const float* m = mass + static_cast<size_t>(plane) * seq_len;
    if (plane % n_kv_heads == 0 && threadIdx.x == 0) dst_lengths[s] = most;
    for (int i = most + threadIdx.x; i < keep; i += kSelectThreads) list[i] = -1;
    if (n <= keep) {
        for (int i = threadIdx.x; i < n; i += kSelectThreads) list[i] = i;
        return;
    }
    const int others = n - recent, want = keep - recent;  // (others > want >= 0)
    for (int i = threadIdx.x; i < recent; i += kSelectThreads) list[want + i] = others + i;
    if (want == 0) return;
    uint32_t prefix = 0, mask = 0;
    int still = want;  // of those whose upper bits are `prefix`, how many are kept
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kSelectThreads) counts[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < others; i += kSelectThreads) {
            const uint32_t key = key_of(m[i]);
            if ((key & mask) == prefix) atomicAdd(&counts[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int above = 0, bin = 255;
            while (above + counts[bin] < still) above += counts[bin--];  // (the counts add up to `still` at least)
            found_bin = bin;
            found_above = above;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(found_bin) << shift;
        mask |= 255u << shift;
        still -= found_above;
        __syncthreads();
    }
    // `prefix` is the smallest weight kept; of those that have it, the first `still` positions.
    int kept_before = 0, equal_before = 0;
    for (int base = 0; base < others; base += kSelectThreads) {
        const int i = base + threadIdx.x;
        const uint32_t key = i < others ? key_of(m[i]) : 0u;
        const bool over = i < others && key > prefix, equal = i < others && key == prefix;
        const unsigned long long below = (1ull << lane) - 1ull;
        const unsigned long long overs = __builtin_amdgcn_ballot_w64(over), equals = __builtin_amdgcn_ballot_w64(equal);
        if (lane == 0) {
            wave_counts[0][wave] = __popcll(overs);
            wave_counts[1][wave] = __popcll(equals);
        }
        __syncthreads();
        int over_at = 0, equal_at = equal_before, over_all = 0, equal_all = 0;
        for (int w = 0; w < kSelectWaves; ++w) {
            if (w < wave) {
                over_at += wave_counts[0][w];
                equal_at += wave_counts[1][w];
            }
            over_all += wave_counts[0][w];
            equal_all += wave_counts[1][w];
        }
        over_at += __popcll(overs & below);
        equal_at += __popcll(equals & below);
        // before position i: over_at larger ones in this stretch, and as many equal ones as are kept
        const int equal_kept_here = min(equal_at, still) - min(equal_before, still);
        if (over || (equal && equal_at < still)) list[kept_before + over_at + equal_kept_here] = i;
        kept_before += over_all + min(equal_before + equal_all, still) - min(equal_before, still);
        equal_before += equal_all;
        __syncthreads();
    }
}

// Rows of the list, 16 bytes a thread: per row head_size / 32 pieces of K codes, as many of V codes, then one thread each for the
// scales of K and V and the weight.  blockIdx.y: sequences and KV heads.
constexpr int kMoveThreads = 256;
template <int kHs>
__global__ __launch_bounds__(kMoveThreads) void move_kernel(Kv4Layer to, float* __restrict__ to_mass, const int* __restrict__ kept, Kv4Layer from,
                                                            const float* __restrict__ from_mass, int planes, int to_len, int from_len, int keep) {
    constexpr int kPieces = kHs / 32;
    const long long i = static_cast<long long>(blockIdx.x) * kMoveThreads + threadIdx.x;
    const int row = static_cast<int>(i / (2 * kPieces + 2)), piece = static_cast<int>(i % (2 * kPieces + 2));
    if (row >= to_len) return;
    for (int plane = blockIdx.y; plane < planes; plane += gridDim.y) {
        const int source = row < keep ? kept[static_cast<size_t>(plane) * keep + row] : -1;
        const size_t dst = static_cast<size_t>(plane) * to_len + row;
        if (source < 0) {
            if (piece == 0) to_mass[dst] = 0.0f;
            continue;
        }
        const size_t src = static_cast<size_t>(plane) * from_len + source;
        if (piece < 2 * kPieces) {
            const int which = piece / kPieces, part = piece % kPieces;
            reinterpret_cast<uintx4*>(to.codes[which])[dst * kPieces + part] = reinterpret_cast<const uintx4*>(from.codes[which])[src * kPieces + part];
            if (piece == 0) to_mass[dst] = from_mass[src];
        } else {
            const int which = piece - 2 * kPieces;
            for (int g = 0; g < kPieces; ++g) to.scales[which][dst * kPieces + g] = from.scales[which][src * kPieces + g];
        }
    }
}

}  // namespace
}  // namespace lpp

extern "C" {

lpp_status lpp_kv4_bytes(const lpp_kv4_shape* shape, size_t* bytes) {
    using namespace lpp;
    LPP_TRY(kv4_check_shape("lpp_kv4_bytes", shape));
    LPP_REQUIRE(bytes != nullptr, "lpp_kv4_bytes: null output");
    *bytes = kv4_bytes(*shape);
    return LPP_OK;
}

lpp_status lpp_kv4_store(void* d_cache, const lpp_kv4_shape* shape, int layer, const void* d_k, const void* d_v, int type, int kv_stride,
                         const int* d_offsets, int n_tokens, const int* d_starts) {
    using namespace lpp;
    LPP_TRY(kv4_check_cache("lpp_kv4_store", d_cache, shape, layer));
    LPP_REQUIRE(type == LPP_F32 || type == LPP_F16, "lpp_kv4_store: type = %d", type);
    LPP_REQUIRE(n_tokens >= 0, "lpp_kv4_store: n_tokens = %d", n_tokens);
    LPP_REQUIRE(d_offsets != nullptr || n_tokens % shape->n_seqs == 0, "lpp_kv4_store: n_tokens = %d is no multiple of n_seqs = %d, and there are no offsets",
                n_tokens, shape->n_seqs);
    const long long kv_dim = static_cast<long long>(shape->n_kv_heads) * shape->head_size;
    LPP_REQUIRE(kv_stride >= kv_dim, "lpp_kv4_store: kv_stride = %d is less than a row of %lld", kv_stride, kv_dim);
    if (n_tokens == 0) return LPP_OK;
    LPP_REQUIRE(d_k && d_v, "lpp_kv4_store: null pointer");
    const int per16 = type == LPP_F32 ? 4 : 8;
    LPP_REQUIRE(reinterpret_cast<uintptr_t>(d_k) % 16 == 0 && reinterpret_cast<uintptr_t>(d_v) % 16 == 0 && kv_stride % per16 == 0,
                "lpp_kv4_store: rows of K and V must start at multiples of 16 bytes");
    const Kv4Layer to = kv4_layer(d_cache, *shape, layer);
    const dim3 grid((static_cast<unsigned>(n_tokens) + 1) / 2);
    if (type == LPP_F32)
        hipLaunchKernelGGL((store_kernel<float>), grid, dim3(kStoreThreads), 0, stream(), to, static_cast<const float*>(d_k), static_cast<const float*>(d_v),
                           kv_stride, d_offsets, d_starts, n_tokens, shape->n_seqs, shape->n_kv_heads, shape->head_size, shape->seq_len);
    else
        hipLaunchKernelGGL((store_kernel<dev::half_t>), grid, dim3(kStoreThreads), 0, stream(), to, static_cast<const dev::half_t*>(d_k),
                           static_cast<const dev::half_t*>(d_v), kv_stride, d_offsets, d_starts, n_tokens, shape->n_seqs, shape->n_kv_heads,
                           shape->head_size, shape->seq_len);
    LPP_CHECK_LAUNCH("store_kernel");
    return LPP_OK;
}

lpp_status lpp_kv4_load(lpp_half* d_k, lpp_half* d_v, const void* d_cache, const lpp_kv4_shape* shape, int layer, int first, int count) {
    using namespace lpp;
    LPP_TRY(kv4_check_cache("lpp_kv4_load", d_cache, shape, layer));
    LPP_REQUIRE(first >= 0 && count >= 0 && first <= shape->seq_len - count, "lpp_kv4_load: positions %d .. + %d of %d", first, count, shape->seq_len);
    if (count == 0) return LPP_OK;
    LPP_REQUIRE(d_k && d_v, "lpp_kv4_load: null pointer");
    LPP_REQUIRE(reinterpret_cast<uintptr_t>(d_k) % 16 == 0 && reinterpret_cast<uintptr_t>(d_v) % 16 == 0,
                "lpp_kv4_load: K and V must start at multiples of 16 bytes");
    const long long planes = static_cast<long long>(shape->n_seqs) * shape->n_kv_heads;
    LPP_REQUIRE(planes <= 0x7fffffffll, "lpp_kv4_load: %lld sequences times KV heads", planes);
    const size_t out_bytes = static_cast<size_t>(planes) * count * shape->head_size * 2;
    LPP_REQUIRE(!ranges_overlap(d_k, out_bytes, d_cache, kv4_bytes(*shape)) && !ranges_overlap(d_v, out_bytes, d_cache, kv4_bytes(*shape)) &&
                    !ranges_overlap(d_k, out_bytes, d_v, out_bytes),
                "lpp_kv4_load: the outputs overlap the cache or each other");
    const int per_head = shape->head_size / 8;
    const size_t words = static_cast<size_t>(count) * per_head;
    const dim3 grid(static_cast<unsigned>((words + kLoadThreads - 1) / kLoadThreads), static_cast<unsigned>(planes < 65535 ? planes : 65535), 2);
    hipLaunchKernelGGL(load_kernel, grid, dim3(kLoadThreads), 0, stream(), reinterpret_cast<dev::half_t*>(d_k), reinterpret_cast<dev::half_t*>(d_v),
                       kv4_layer(d_cache, *shape, layer), static_cast<int>(planes), per_head, shape->seq_len, first, count);
    LPP_CHECK_LAUNCH("load_kernel");
    return LPP_OK;
}

lpp_status lpp_kv4_evict(void* d_dst, const lpp_kv4_shape* dst, int dst_layer, float* d_dst_mass, int* d_dst_lengths, int* d_kept, const void* d_src,
                         const lpp_kv4_shape* src, int src_layer, const float* d_mass, const int* d_lengths, int keep, int recent) {
    using namespace lpp;
    LPP_TRY(kv4_check_cache("lpp_kv4_evict", d_dst, dst, dst_layer));
    LPP_TRY(kv4_check_cache("lpp_kv4_evict", d_src, src, src_layer));
    LPP_REQUIRE(d_dst_mass && d_dst_lengths && d_kept && d_mass && d_lengths, "lpp_kv4_evict: null pointer");
    LPP_REQUIRE(dst->n_seqs == src->n_seqs && dst->n_kv_heads == src->n_kv_heads && dst->head_size == src->head_size,
                "lpp_kv4_evict: the caches are of %d and %d sequences, %d and %d KV heads, heads of %d and %d", dst->n_seqs, src->n_seqs,
                dst->n_kv_heads, src->n_kv_heads, dst->head_size, src->head_size);
    LPP_REQUIRE(recent >= 0 && recent <= keep && keep > 0 && keep <= dst->seq_len, "lpp_kv4_evict: keep = %d, recent = %d, room for %d", keep, recent,
                dst->seq_len);
    const long long planes = static_cast<long long>(dst->n_seqs) * dst->n_kv_heads;
    LPP_REQUIRE(planes <= 0x7fffffffll, "lpp_kv4_evict: %lld sequences times KV heads", planes);
    LPP_REQUIRE(!ranges_overlap(d_dst, kv4_bytes(*dst), d_src, kv4_bytes(*src)), "lpp_kv4_evict: the caches overlap");
    const size_t dst_mass_bytes = kv4_layer_rows(*dst) * dst->n_layers * 4, src_mass_bytes = kv4_layer_rows(*src) * src->n_layers * 4;
    LPP_REQUIRE(!ranges_overlap(d_dst_mass, dst_mass_bytes, d_mass, src_mass_bytes), "lpp_kv4_evict: d_dst_mass overlaps d_mass");
    LPP_REQUIRE(!ranges_overlap(d_dst_lengths, 4 * static_cast<size_t>(dst->n_seqs), d_lengths, 4 * static_cast<size_t>(dst->n_seqs)),
                "lpp_kv4_evict: d_dst_lengths overlaps d_lengths");
    float* dst_mass = d_dst_mass + kv4_layer_rows(*dst) * dst_layer;
    const float* src_mass = d_mass + kv4_layer_rows(*src) * src_layer;
    hipLaunchKernelGGL(select_kernel, dim3(static_cast<unsigned>(planes)), dim3(kSelectThreads), 0, stream(), d_kept, d_dst_lengths, src_mass, d_lengths,
                       dst->n_kv_heads, src->seq_len, keep, recent);
    LPP_CHECK_LAUNCH("select_kernel");
    const Kv4Layer to = kv4_layer(d_dst, *dst, dst_layer), from = kv4_layer(d_src, *src, src_layer);
    const long long threads = static_cast<long long>(dst->seq_len) * (2 * dst->head_size / 32 + 2);
    const dim3 grid(static_cast<unsigned>((threads + kMoveThreads - 1) / kMoveThreads), static_cast<unsigned>(planes < 65535 ? planes : 65535));
    if (dst->head_size == 64)
        hipLaunchKernelGGL((move_kernel<64>), grid, dim3(kMoveThreads), 0, stream(), to, dst_mass, d_kept, from, src_mass, static_cast<int>(planes),
                           dst->seq_len, src->seq_len, keep);
    else
        hipLaunchKernelGGL((move_kernel<128>), grid, dim3(kMoveThreads), 0, stream(), to, dst_mass, d_kept, from, src_mass, static_cast<int>(planes),
                           dst->seq_len, src->seq_len, keep);
    LPP_CHECK_LAUNCH("move_kernel");
    return LPP_OK;
}

}  // extern "C"
