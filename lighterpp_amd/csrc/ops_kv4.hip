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

// A word of the codes of eight values: the integers nearest to (x - low) / scale, in 0 .. 15.  In fp32, as fifteen times a number that is cut to 0 ..
// 1 as it is formed, the quotient is off by less than 15 * 4 * 2^-24 and by 2^-22 of low / scale; a word with a quotient nearer than that to a border
// (within 1e-5 and 2^-21) is formed again by the sign of x - low - border * scale.  (Of fp32 values that is one word in 6000; binary16 values lie on
// a border itself often, about one word in 300.)  Adding 2^23 rounds to the nearest integer, ties to even, and leaves it in the lowest bits: the
// codes are added up with what is above them, which is taken off at the end.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float low, float scale) {
    const float inverse = scale > 0.0f ? __builtin_amdgcn_rcpf(scale) : 0.0f;
    const float slope = inverse * (1.0f / 15.0f), shift = -low * slope;
    uint32_t word = 0, above = 0;
    float furthest = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float t = __builtin_amdgcn_fmed3f(fmaf(x[e], slope, shift), 0.0f, 1.0f), shifted = fmaf(t, 15.0f, 8388608.0f);
        furthest = fmaxf(furthest, fabsf(fmaf(t, 15.0f, 8388608.0f - shifted)));
        word += __float_as_uint(shifted) << (4 * (e / 2) + 16 * (e & 1));
        above += 0x4B000000u << (4 * (e / 2) + 16 * (e & 1));
    }
    word -= above;
    if (furthest > 0.5f - 1e-5f - fabsf(low * inverse) * 0x1p-21f) {
#pragma clang fp contract(off)
        word = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // difference + left is x - low; the border between f and f + 1 (an f one off near an integer decides the same)
            const float difference = x[e] - low, taken = difference - x[e], left = (x[e] - (difference - taken)) + (-low - taken);
            const float f = floorf(__builtin_amdgcn_fmed3f(difference * inverse, 0.0f, 14.0f));
            const float beyond = fmaf(-(f + 0.5f), scale, difference) + left;
            const uint32_t below = static_cast<uint32_t>(f);
            word |= (below + (beyond > 0.0f || (beyond == 0.0f && (below & 1u)) ? 1u : 0u)) << (4 * (e / 2) + 16 * (e & 1));
        }
    }
    return word;
}

// The product is hidden from the compiler, which would otherwise form it and its rounding to binary16 in one instruction, with one rounding.
__device__ __forceinline__ float fifteenth(float r) {
    float product = r * (1.0f / 15.0f);
    asm("" : "+v"(product));
    return product;
}

// One wavefront per row, K and V; a lane has a word's eight values, two words of each at a time.  The first values are requested along with the
// sequences' ends and starts, before anything is known about the row: what a row takes is the time of its requests, one after the other.
// 14208 rows of 8 heads of 128, binary16: 25.6 us, 3.0 TB/s of values read and codes written; 16 rows of 8 heads of 64 3.3 us.
template <typename T>
__global__ __launch_bounds__(kStoreThreads) void store_kernel(Kv4Layer to, const T* __restrict__ k, const T* __restrict__ v, int stride,
                                                              const int* __restrict__ offsets, const int* __restrict__ starts, int n_tokens,
                                                              int n_seqs, int n_kv_heads, int head_size, int seq_len) {
    constexpr int kAtOnce = 2, kLoads = sizeof(T) / 2;  // words; requests of 16 bytes to a word
    const int lane = lane_id();
    const int row = static_cast<int>(blockIdx.x) * (kStoreThreads / kWave) + wave_index();
    if (row >= n_tokens) return;
    const T* from[2] = {k + static_cast<size_t>(row) * stride, v + static_cast<size_t>(row) * stride};
    const int words = n_kv_heads * head_size / 8, per_head = head_size / 8;
    uintx4 raw[2][kAtOnce][kLoads];
    auto request = [&](int w0) {
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int w = min(w0 + kWave * u + lane, words - 1);
#pragma unroll
                for (int i = 0; i < kLoads; ++i) raw[which][u][i] = load16(from[which] + 8 * w + 8 / kLoads * i);
            }
    };
    request(0);
    int s = 0, first = 0, start = 0;
    if (offsets != nullptr && n_seqs > kWave) {
        s = count_up_to(n_seqs, row, [&](int at) { return offsets[at + 1]; });
        if (s >= n_seqs) return;
        first = max(offsets[s], 0);
        if (row < first) return;
        if (starts != nullptr) start = starts[s];
    } else if (offsets != nullptr) {
        const int at = min(lane, n_seqs - 1);
        const int begin = offsets[0], end = offsets[at + 1], its_start = starts != nullptr ? starts[at] : 0;
        s = __popcll(__builtin_amdgcn_ballot_w64(end <= row && lane < n_seqs));
        if (s >= n_seqs) return;
        first = max(s > 0 ? __builtin_amdgcn_readlane(end, s > 0 ? s - 1 : 0) : begin, 0);
        if (row < first) return;
        start = __builtin_amdgcn_readlane(its_start, s);
    } else {
        const int each = n_tokens / n_seqs;
        s = row / each;
        first = s * each;
        if (starts != nullptr) start = starts[s];
    }
    const long long pos = static_cast<long long>(start) + row - first;
    if (pos < 0 || pos >= seq_len) return;
    const int shift = per_head == 8 ? 3 : 4;
    const size_t base = static_cast<size_t>(s) * n_kv_heads * seq_len + static_cast<size_t>(pos);
    for (int w0 = 0; w0 < words; w0 += kAtOnce * kWave) {
        float x[2][kAtOnce][8];
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (kLoads == 1) x[which][u][e] = static_cast<float>(as_half8(raw[which][u][0])[e]);
                    else x[which][u][e] = as_float4(raw[which][u][e / 4])[e & 3];
                }
        if (w0 + kAtOnce * kWave < words) request(w0 + kAtOnce * kWave);
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const float(&mine)[8] = x[which][u];
                const int w = w0 + kWave * u + lane;
                float least = mine[0], most = mine[0];
                uint32_t size = 0;  // (as an integer: NaN is the largest)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    least = fminf(least, mine[e]);
                    most = fmaxf(most, mine[e]);
                    size = max(size, __float_as_uint(mine[e]) << 1);
                }
                least = quad_min(least);
                most = quad_max(most);
                const int bad = quad_or(size > (__float_as_uint(32768.0f) << 1) ? 1 : 0);
                const half_t low16 = static_cast<half_t>(least), scale16 = static_cast<half_t>(fifteenth(most - least));
                uint32_t word = 0, pair = 0x7E000000u;
                if (!bad) {
                    word = codes_of(mine, static_cast<float>(low16), static_cast<float>(scale16));
                    pair = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, scale16)) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, low16)) << 16;
                }
                // (a row's words are whole groups, so a group's four lanes are all within or all beyond it)
                if (w < words) {
                    const int head = w >> shift, in_head = w & (per_head - 1);
                    const size_t at = base + static_cast<size_t>(head) * seq_len;
                    to.codes[which][at * per_head + in_head] = word;
                    if ((w & 3) == 0) to.scales[which][at * (per_head / 4) + in_head / 4] = pair;
                }
            }
    }
}

// One thread per word; blockIdx.y: sequences and KV heads, blockIdx.z: K, V.  Bound by what it writes: 6 x 8 heads of 128, 4000 positions: 24 us,
// 5.4 TB/s.
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

// One workgroup per sequence and KV head: the keep - recent positions of largest weight among the first n - recent, then the list in order. The
// smallest weight kept is found by its bits, 11, 11 and 10 at a time from the top: counts of every value of those bits among the weights that agree
// with what is known, added up from above.  A thread holds kHeld weights in registers (kOnce: all it has; else stretches of them, read again in every
// pass).  A sequence and KV head of 2048 positions: 7.7 us, 128 of up to 8100 11 us, the time of its passes one after the other; fewer threads are no
// faster.
constexpr int kBins = 2048;
template <int kHeld, bool kOnce>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(int* __restrict__ kept, int* __restrict__ dst_lengths, const float* __restrict__ mass,
                                                                const int* __restrict__ lengths, int n_kv_heads, int seq_len, int keep, int recent) {
    constexpr int kStretch = kHeld * kSelectThreads, kPerThread = kBins / kSelectThreads;
    __shared__ int counts[kBins];
    __shared__ int wave_counts[kHeld * kSelectWaves], wave_equals[kHeld * kSelectWaves];
    __shared__ int wave_sums[kSelectWaves];
    __shared__ int found_bin, found_above;
    const int plane = blockIdx.x, s = plane / n_kv_heads, lane = lane_id(), wave = wave_index(), thread = threadIdx.x;
    const int n = min(max(lengths[s], 0), seq_len), most = min(n, keep);
    int* list = kept + static_cast<size_t>(plane) * keep;
    const float* m = mass + static_cast<size_t>(plane) * seq_len;
    if (plane % n_kv_heads == 0 && thread == 0) dst_lengths[s] = most;
    for (int i = most + thread; i < keep; i += kSelectThreads) list[i] = -1;
    if (n <= keep) {
        for (int i = thread; i < n; i += kSelectThreads) list[i] = i;
        return;
    }
    const int others = n - recent, want = keep - recent;  // (others > want >= 0)
    for (int i = thread; i < recent; i += kSelectThreads) list[want + i] = others + i;
    if (want == 0) return;
    uint32_t keys[kHeld];
    auto read = [&](int base) {
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = base + j * kSelectThreads + thread;
            keys[j] = __float_as_uint(m[min(i, others - 1)]);
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j) keys[j] = key_of(__uint_as_float(keys[j]));
    };
    // (positions at or behind `others` are those whose number says so)
    if constexpr (kOnce) read(0);
    uint32_t prefix = 0, mask = 0;
    int still = want;  // of those whose upper bits are `prefix`, how many are kept
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) counts[i * kSelectThreads + thread] = 0;
        __syncthreads();
        for (int base = 0; base < others; base += kStretch) {
            if constexpr (!kOnce) read(base);
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if (base + j * kSelectThreads + thread < others && (keys[j] & mask) == prefix) atomicAdd(&counts[(keys[j] >> shift) & digits], 1);
        }
        __syncthreads();
        // thread t has bins kBins - 1 - kPerThread t and below: sums from above
        int mine[kPerThread], sum = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            mine[i] = counts[kBins - 1 - kPerThread * thread - i];
            sum += mine[i];
        }
        const int upto = wave_inclusive_sum(sum);
        if (lane == kWave - 1) wave_sums[wave] = upto;
        __syncthreads();
        int above = upto - sum;
        for (int w = 0; w < wave; ++w) above += wave_sums[w];
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            if (above < still && above + mine[i] >= still) {  // (one bin of one thread)
                found_bin = kBins - 1 - kPerThread * thread - i;
                found_above = above;
            }
            above += mine[i];
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(found_bin) << shift;
        mask |= digits << shift;
        still -= found_above;
        // (found_bin is written again after two barriers)
    }
    // `prefix` is the smallest weight kept; of those that have it, the first `still` positions.  Counts of every 64 positions, added up in order.
    int kept_before = 0, equal_before = 0;
    const unsigned long long below = (1ull << lane) - 1ull;
    for (int base = 0; base < others; base += kStretch) {
        if constexpr (!kOnce) read(base);
        unsigned long long overs[kHeld], equals[kHeld];
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const bool there = base + j * kSelectThreads + thread < others;
            overs[j] = __builtin_amdgcn_ballot_w64(there && keys[j] > prefix);
            equals[j] = __builtin_amdgcn_ballot_w64(there && keys[j] == prefix);
            if (lane == 0) {
                wave_counts[j * kSelectWaves + wave] = __popcll(overs[j]);
                wave_equals[j * kSelectWaves + wave] = __popcll(equals[j]);
            }
        }
        __syncthreads();
        // every wavefront adds all of them up by itself, 64 at a time, and keeps what is before its own
        int over_at[kHeld], equal_at[kHeld], over_all = 0, equal_all = 0;
#pragma unroll
        for (int j0 = 0; j0 < kHeld; j0 += kWave / kSelectWaves) {
            const int at = j0 * kSelectWaves + lane;
            const int over = at < kHeld * kSelectWaves ? wave_counts[at] : 0, equal = at < kHeld * kSelectWaves ? wave_equals[at] : 0;
            const int over_upto = wave_inclusive_sum(over), equal_upto = wave_inclusive_sum(equal);
#pragma unroll
            for (int j = j0; j < j0 + kWave / kSelectWaves && j < kHeld; ++j) {
                const int me = (j - j0) * kSelectWaves + wave;
                over_at[j] = over_all + __builtin_amdgcn_readlane(over_upto - over, me);
                equal_at[j] = equal_all + __builtin_amdgcn_readlane(equal_upto - equal, me);
            }
            over_all += __builtin_amdgcn_readlane(over_upto, kWave - 1);
            equal_all += __builtin_amdgcn_readlane(equal_upto, kWave - 1);
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int equal_rank = equal_before + equal_at[j] + __popcll(equals[j] & below);
            const int at = kept_before + over_at[j] + __popcll(overs[j] & below) + min(equal_rank, still) - min(equal_before, still);
            const bool over = (overs[j] >> lane) & 1ull, equal = (equals[j] >> lane) & 1ull;
            if (over || (equal && equal_rank < still)) list[at] = base + j * kSelectThreads + thread;
        }
        kept_before += over_all + min(equal_before + equal_all, still) - min(equal_before, still);
        equal_before += equal_all;
        if constexpr (!kOnce) __syncthreads();
    }
}

// Rows of the list.  A block has kMovePieces pieces of one part of the cache, one behind the other: 16 bytes of codes of K or V (first
// blocks, `code_blocks` each), or a row's scales of K and V and its weight.  blockIdx.y: sequences and KV heads.  128 of them, 2000 rows
// kept of heads of 128 each: 28 us, 2.9 TB/s read and written.
constexpr int kMoveThreads = 256, kMoveEach = 4, kMovePieces = kMoveThreads * kMoveEach;
template <int kHs>
__global__ __launch_bounds__(kMoveThreads) void move_kernel(Kv4Layer to, float* __restrict__ to_mass, const int* __restrict__ kept, Kv4Layer from,
                                                            const float* __restrict__ from_mass, int planes, int to_len, int from_len, int keep,
                                                            int code_blocks) {
    constexpr unsigned kCodes = kHs / 32, kWords = kHs / kKv4Group;
    typedef uint32_t Scales __attribute__((ext_vector_type(kWords)));
    const int block = blockIdx.x;
    for (int plane = blockIdx.y; plane < planes; plane += gridDim.y) {
        const size_t dst = static_cast<size_t>(plane) * to_len, src = static_cast<size_t>(plane) * from_len;
        const int* list = kept + static_cast<size_t>(plane) * keep;
        int source[kMoveEach];
        if (block < 2 * code_blocks) {
            const int which = block >= code_blocks;
            const unsigned first = static_cast<unsigned>(which ? block - code_blocks : block) * kMovePieces + threadIdx.x;
            const uintx4* in = reinterpret_cast<const uintx4*>(from.codes[which]) + src * kCodes;
            uintx4* out = reinterpret_cast<uintx4*>(to.codes[which]) + dst * kCodes;
            uintx4 x[kMoveEach];
#pragma unroll
            for (int u = 0; u < kMoveEach; ++u) {
                const unsigned row = (first + kMoveThreads * u) / kCodes;
                source[u] = row < static_cast<unsigned>(keep) ? list[row] : -1;
            }
#pragma unroll
            for (int u = 0; u < kMoveEach; ++u) x[u] = in[static_cast<size_t>(max(source[u], 0)) * kCodes + (first + kMoveThreads * u) % kCodes];
#pragma unroll
            for (int u = 0; u < kMoveEach; ++u)
                if (source[u] >= 0) out[first + kMoveThreads * u] = x[u];
        } else {
            const unsigned first = static_cast<unsigned>(block - 2 * code_blocks) * kMovePieces + threadIdx.x;
            Scales x[2][kMoveEach];
            float w[kMoveEach];
#pragma unroll
            for (int u = 0; u < kMoveEach; ++u) source[u] = first + kMoveThreads * u < static_cast<unsigned>(keep) ? list[first + kMoveThreads * u] : -1;
#pragma unroll
            for (int u = 0; u < kMoveEach; ++u) {
                const size_t at = src + max(source[u], 0);
                x[0][u] = reinterpret_cast<const Scales*>(from.scales[0])[at];
                x[1][u] = reinterpret_cast<const Scales*>(from.scales[1])[at];
                w[u] = from_mass[at];
            }
#pragma unroll
            for (int u = 0; u < kMoveEach; ++u) {
                const unsigned row = first + kMoveThreads * u;
                if (source[u] >= 0) {
                    reinterpret_cast<Scales*>(to.scales[0])[dst + row] = x[0][u];
                    reinterpret_cast<Scales*>(to.scales[1])[dst + row] = x[1][u];
                }
                if (row < static_cast<unsigned>(to_len)) to_mass[dst + row] = source[u] >= 0 ? w[u] : 0.0f;
            }
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
    const unsigned blocks = (static_cast<unsigned>(n_tokens) + kStoreThreads / dev::kWave - 1) / (kStoreThreads / dev::kWave);
    LPP_REQUIRE(static_cast<long long>(blocks) * kStoreThreads < (1ll << 32), "lpp_kv4_store: n_tokens = %d are too many for a launch", n_tokens);
    LPP_REQUIRE(d_k && d_v, "lpp_kv4_store: null pointer");
    const int per16 = type == LPP_F32 ? 4 : 8;
    LPP_REQUIRE(reinterpret_cast<uintptr_t>(d_k) % 16 == 0 && reinterpret_cast<uintptr_t>(d_v) % 16 == 0 && kv_stride % per16 == 0,
                "lpp_kv4_store: rows of K and V must start at multiples of 16 bytes");
    const size_t in_bytes = (static_cast<size_t>(n_tokens - 1) * kv_stride + kv_dim) * (type == LPP_F32 ? 4 : 2);
    LPP_REQUIRE(!ranges_overlap(d_k, in_bytes, d_cache, kv4_bytes(*shape)) && !ranges_overlap(d_v, in_bytes, d_cache, kv4_bytes(*shape)),
                "lpp_kv4_store: the rows overlap the cache");
    const size_t seqs_bytes = static_cast<size_t>(shape->n_seqs) * 4;
    LPP_REQUIRE((d_offsets == nullptr || !ranges_overlap(d_offsets, seqs_bytes + 4, d_cache, kv4_bytes(*shape))) &&
                    (d_starts == nullptr || !ranges_overlap(d_starts, seqs_bytes, d_cache, kv4_bytes(*shape))),
                "lpp_kv4_store: d_offsets or d_starts overlaps the cache");
    const Kv4Layer to = kv4_layer(d_cache, *shape, layer);
    const dim3 grid(blocks);
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
    LPP_REQUIRE(planes * kSelectThreads < (1ll << 32), "lpp_kv4_evict: %lld sequences times KV heads", planes);
    const struct {
        const char* name;
        const void* at;
        size_t bytes;
    } buffers[] = {{"d_dst", d_dst, kv4_bytes(*dst)},
                   {"d_dst_mass", d_dst_mass, kv4_layer_rows(*dst) * dst->n_layers * 4},
                   {"d_dst_lengths", d_dst_lengths, 4 * static_cast<size_t>(dst->n_seqs)},
                   {"d_kept", d_kept, 4 * static_cast<size_t>(planes) * keep},
                   {"d_src", d_src, kv4_bytes(*src)},
                   {"d_mass", d_mass, kv4_layer_rows(*src) * src->n_layers * 4},
                   {"d_lengths", d_lengths, 4 * static_cast<size_t>(src->n_seqs)}};
    for (int a = 0; a < 4; ++a)  // (what is written, and all behind it)
        for (int b = a + 1; b < 7; ++b)
            LPP_REQUIRE(!ranges_overlap(buffers[a].at, buffers[a].bytes, buffers[b].at, buffers[b].bytes), "lpp_kv4_evict: %s overlaps %s", buffers[a].name,
                        buffers[b].name);
    float* dst_mass = d_dst_mass + kv4_layer_rows(*dst) * dst_layer;
    const float* src_mass = d_mass + kv4_layer_rows(*src) * src_layer;
    const auto select = src->seq_len <= 4 * kSelectThreads    ? &select_kernel<4, true>
                        : src->seq_len <= 8 * kSelectThreads  ? &select_kernel<8, true>
                        : src->seq_len <= 32 * kSelectThreads ? &select_kernel<32, true>
                                                              : &select_kernel<32, false>;
    hipLaunchKernelGGL(select, dim3(static_cast<unsigned>(planes)), dim3(kSelectThreads), 0, stream(), d_kept, d_dst_lengths, src_mass, d_lengths,
                       dst->n_kv_heads, src->seq_len, keep, recent);
    LPP_CHECK_LAUNCH("select_kernel");
    const Kv4Layer to = kv4_layer(d_dst, *dst, dst_layer), from = kv4_layer(d_src, *src, src_layer);
    const auto blocks_of = [](long long pieces) { return static_cast<int>((pieces + kMovePieces - 1) / kMovePieces); };
    const int code_blocks = blocks_of(static_cast<long long>(keep) * (dst->head_size / 32));
    const dim3 grid(2 * code_blocks + blocks_of(dst->seq_len), static_cast<unsigned>(planes < 65535 ? planes : 65535));
    hipLaunchKernelGGL((dst->head_size == 64 ? &move_kernel<64> : &move_kernel<128>), grid, dim3(kMoveThreads), 0, stream(), to, dst_mass, d_kept, from,
                       src_mass, static_cast<int>(planes), dst->seq_len, src->seq_len, keep, code_blocks);
    LPP_CHECK_LAUNCH("move_kernel");
    return LPP_OK;
}

}  // extern "C"
