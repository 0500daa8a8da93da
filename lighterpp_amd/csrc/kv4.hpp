// kv4.hpp -- the cache of 4 bits: where its parts lie, what a word of codes
// stands for, and the checks its entry points share.
#pragma once

#include "lpp_device.hpp"
#include "lpp_internal.hpp"

namespace lpp {

constexpr int kKv4Group = 32;             // values that share a scale
constexpr int kKv4MaxSeqLen = 1 << 24;    // a head's rows stay within 31 bits of bytes
constexpr int kMaxSharedHeads = 16;       // query heads to a KV head

// One layer of a cache: rows of its four parts, [sequence][KV head][position].
struct Kv4Layer {
    uint32_t* codes[2];   // K, V: head_size / 8 words a row
    uint32_t* scales[2];  // head_size / 32 words a row: scale in the low half, lowest value in the high half
};

inline size_t kv4_layer_rows(const lpp_kv4_shape& s) { return static_cast<size_t>(s.n_seqs) * s.n_kv_heads * s.seq_len; }

inline Kv4Layer kv4_layer(const void* cache, const lpp_kv4_shape& s, int layer) {
    const size_t rows = kv4_layer_rows(s) * s.n_layers, before = kv4_layer_rows(s) * layer;
    const size_t code_words = s.head_size / 8, scale_words = s.head_size / kKv4Group;
    uint32_t* base = const_cast<uint32_t*>(static_cast<const uint32_t*>(cache));
    Kv4Layer l;
    l.codes[0] = base + before * code_words;
    l.codes[1] = base + (rows + before) * code_words;
    l.scales[0] = base + 2 * rows * code_words + before * scale_words;
    l.scales[1] = base + 2 * rows * code_words + (rows + before) * scale_words;
    return l;
}

inline size_t kv4_bytes(const lpp_kv4_shape& s) { return kv4_layer_rows(s) * s.n_layers * s.head_size / 4 * 5; }

// (the product of the counts fits 40 bits, and so every offset 64)
inline lpp_status kv4_check_shape(const char* who, const lpp_kv4_shape* s) {
    LPP_REQUIRE(s != nullptr, "%s: null shape", who);
    LPP_REQUIRE(s->n_layers > 0 && s->n_seqs > 0 && s->n_kv_heads > 0 && s->seq_len > 0,
                "%s: n_layers = %d, n_seqs = %d, n_kv_heads = %d, seq_len = %d", who, s->n_layers, s->n_seqs, s->n_kv_heads, s->seq_len);
    LPP_REQUIRE(s->head_size == 64 || s->head_size == 128, "%s: head_size = %d is neither 64 nor 128", who, s->head_size);
    LPP_REQUIRE(s->seq_len <= kKv4MaxSeqLen, "%s: seq_len = %d beyond %d", who, s->seq_len, kKv4MaxSeqLen);
    const double rows = static_cast<double>(s->n_layers) * s->n_seqs * s->n_kv_heads * s->seq_len;
    LPP_REQUIRE(rows <= 1099511627776.0, "%s: %.0f rows are beyond 2^40", who, rows);
    return LPP_OK;
}
inline lpp_status kv4_check_cache(const char* who, const void* cache, const lpp_kv4_shape* s, int layer) {
    LPP_TRY(kv4_check_shape(who, s));
    LPP_REQUIRE(cache != nullptr, "%s: null cache", who);
    LPP_REQUIRE(reinterpret_cast<uintptr_t>(cache) % 16 == 0, "%s: the cache is not 16-byte aligned", who);
    LPP_REQUIRE(layer >= 0 && layer < s->n_layers, "%s: layer = %d outside [0, %d)", who, layer, s->n_layers);
    return LPP_OK;
}

inline bool ranges_overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

// A kernel's LDS need, told to the runtime once per device (the attribute belongs to the device's copy of the kernel).
inline lpp_status tell_lds(const void* kernel, int bytes, bool (&told)[64]) {
    int device = 0;
    LPP_HIP(hipGetDevice(&device));
    if (device < 0 || device >= 64 || !told[device]) {
        LPP_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (device >= 0 && device < 64) told[device] = true;
    }
    return LPP_OK;
}

namespace dev {

// A softmax in one walk takes its weights as 2^(score - reference).  The reference lies kLift below a score of the row and moves when a score passes that
// one by more than kSlack: the largest weight is between 2^8 and 2^15, near binary16's largest, so that small ones keep bits in its subnormals (2^-33
// of the largest weight, head and remainder).
constexpr float kLift = 9.0f, kSlack = 6.0f;

// The eight binary16 numbers that a word of codes stands for.  A code in the last bits of a half whose exponent is that of 1024 is
// 1024 + code, four bits further up and with the exponent of 64 it is 64 + code: a pair costs one and-or, one (exact) subtraction and one
// fused multiply-add, the one rounding, and a word one shift.
struct Kv4Reader {
    // (in vector registers: v_and_or_b32 takes one constant from a scalar register, the other would make it two instructions)
    uint32_t as1024 = 0x64006400u, as64 = 0x54005400u;
    __device__ __forceinline__ Kv4Reader() { asm("" : "+v"(as1024), "+v"(as64)); }
    __device__ __forceinline__ half8_t operator()(uint32_t codes, uint32_t scale_and_low) const {
        const half2_t both = __builtin_bit_cast(half2_t, scale_and_low);
        const half2_t scale = {both[0], both[0]}, low = {both[1], both[1]};
        const half_t k1024 = static_cast<half_t>(1024.0f), k64 = static_cast<half_t>(64.0f);
        const uint32_t upper = codes >> 8;
        half8_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t from = i < 2 ? codes : upper;
            const uint32_t bits = (i & 1) ? (from & 0x00F000F0u) | as64 : (from & 0x000F000Fu) | as1024;
            const half2_t base = (i & 1) ? half2_t{k64, k64} : half2_t{k1024, k1024};
            const half2_t pair = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, bits) - base, scale, low);
            v[2 * i] = pair[0];
            v[2 * i + 1] = pair[1];
        }
        return v;
    }
};

// v + that of the same lane of the wavefront's other half.
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum over the wavefront's lanes up to and with this one.
__device__ __forceinline__ int wave_inclusive_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr by 1, 2, 4, 8: zero comes in
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = r0 + __builtin_amdgcn_readlane(v, 31), r2 = r1 + __builtin_amdgcn_readlane(v, 47);
    const int row = lane_id() >> 4;
    return v + (row == 0 ? 0 : row == 1 ? r0 : row == 2 ? r1 : r2);
}

// How many of n values that do not decrease, value(0) .. value(n - 1), are at or below `limit`.  The whole wavefront looks at 64 of them at a time:
// one round for up to 64, two for 4096.
template <typename Value>
__device__ __forceinline__ int count_up_to(int n, int limit, Value value) {
    int from = 0, count = n;  // the first `from` are; none behind the first from + count is
    while (count > 0) {
        const int step = (count + kWave - 1) / kWave, at = from + step * lane_id() + step - 1;
        const bool is = at < from + count && value(at) <= limit;
        const int blocks = __popcll(__builtin_amdgcn_ballot_w64(is));
        const int left = count - step * blocks;
        from += step * blocks;
        count = step == 1 ? 0 : min(left, step - 1);
        if (blocks == kWave) break;
    }
    return from;
}

}  // namespace dev
}  // namespace lpp
