// ops_prompt.hip -- lpp_prompt_attention: causal attention of whole prompts,
// packed one behind the other.
//
// out[t] = sum_p w(t, p) v[p] / sum_p w(t, p) with w(t, p) = 2^(scale q[t] . k[p] - top(t)), over the positions p <= t of t's sequence, scale =
// log2(e) / sqrt(head_size).  One walk over the positions: `top` lies kLift below a score of the row so far, and moves (sum and output are rescaled) only when a
// score passes that one by more than kSlack; any value near the maximum would do, since it cancels.
//
// Both products run on the matrix cores, 32 positions x 32 query rows at a time: scores = K Q^T, whose result has a query row to a lane and its
// positions in that lane's registers, as the second product, V^T W^T, wants its second operand; so weights never leave registers, and maximum and sum
// of a row are two lanes' business.  The order in which the first product's rows come out is made good by the order in which transposing reads take V
// rows from LDS.  Weights enter as binary16 head and remainder, and so do fp32 queries: the second product is twice its size, with fp32 the first too.
// (Weights rounded to binary16 would be enough for binary16 activations by their size, but the output's error would be 2.4e-4 to 2.7e-4 of its norm where
// its own rounding makes 2.0e-4; with the remainders it is rounded once, and is within 2e-5 of fp32 arithmetic rounded.  They cost 4 % with prompts of
// 250 rows, a fifth at 2000 and a third at 8191.)
//
// What bounds it.  A long document (8191 rows, 32 heads of 128 on 8, binary16): 731 to 759 us (machines hold different clocks), 1090 to 1130 TFLOP/s
// of products, where a matrix product of 8192^3 reaches 1186; matrix cores busy 64 % of the cycles, vector ALUs 50 %, LDS 22 %, at the clock of 1.7
// GHz that the power leaves.  Without exponentials, a maximum, or the multiplication by the scale fp32 gained 0 to 10 %; two query tiles to a
// wavefront, for half the reads of LDS, are slower (half the wavefronts: 4096 rows, 32 heads of 64, fp32 224 us for 157; heads of 128 do not fit the
// registers).  Several pages (7 of up to 1500 rows, 32 heads of 64 on 8, fp32): 111 us, of which the remainders' products are a third.  Few rows (4
// of up to 45): 5.9 us, the time of the requests one after the other: offsets, rows, and the write.
#include <type_traits>

#include "kv4.hpp"

namespace lpp {
namespace {

using namespace dev;

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

// A workgroup is kR x kP wavefronts: kR own 32 query rows each, (32 / shared) consecutive tokens x the query heads of one KV head, and share
// the K and V rows of every step of kStep positions; kP take the steps in turn and merge what they have at the end.
template <int kHs, int kR, int kP, int kStepRows>
struct Shape {
    static constexpr int kStep = kStepRows, kRowBytes = 2 * kHs, kPieces = kHs / 8;
    static constexpr int kHalfBytes = kStep * kRowBytes, kStageBytes = 2 * kHalfBytes;  // K rows, then V rows
    static constexpr int kStages = 2;
    static constexpr int kPartFloats = (kHs / 2 + 2) * 64;  // a wavefront's maximum, sum and output
    static constexpr int kMergeBytes = kP > 1 ? kP * kR * kPartFloats * 4 : 0;
    static constexpr int kStepBytes = kP * kStages * kStageBytes;
    static constexpr int kLdsBytes = kStepBytes > kMergeBytes ? kStepBytes : kMergeBytes;
    static_assert(kStageBytes % (1024 * kR) == 0, "every wavefront makes the same number of requests");
    static_assert(kLdsBytes <= 160 * 1024, "LDS of a workgroup");
};

struct PromptJob {
    void* out;
    const void* q;
    const half_t* k;
    const half_t* v;
    const int* offsets;
    int n_seqs, n_tokens, shared, n_kv_heads;
    int q_stride, kv_stride, out_stride;
};

__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int kCount>
__device__ __forceinline__ void wait_requests() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCount) : "memory");
}
__device__ __forceinline__ int wave_sum_int(int v) { return __builtin_amdgcn_readlane(wave_inclusive_sum(v), kWave - 1); }

// The workgroup's tile: which of its sequence's tiles it is, and the sequence's rows (returned; 0: it has none).  Up to 64 sequences: in the order of
// their walks' lengths, longest first, whatever the sequence.  More: sequence s's tiles, the last one first, from number
// offsets[s] / tokens + s on, which leaves room for those of the sequences before (s counts those without rows too, so the numbers run to n_tokens /
// tokens + n_seqs).
__device__ __forceinline__ int find_tile(const PromptJob& job, int tokens, int& tile, int& first_row) {
    if (job.offsets == nullptr) {
        first_row = 0;
        tile = (job.n_tokens + tokens - 1) / tokens - 1 - tile;
        return tile >= 0 ? job.n_tokens : 0;
    }
    const auto offset = [&](int s) { return min(max(job.offsets[s], 0), job.n_tokens); };
    if (job.n_seqs > kWave) {
        const int s = count_up_to(job.n_seqs, tile, [&](int at) { return offset(at) / tokens + at; }) - 1;
        if (s < 0) return 0;
        const int begin = __builtin_amdgcn_readfirstlane(offset(s)), end = __builtin_amdgcn_readfirstlane(offset(s + 1));
        first_row = begin;
        tile = (end - begin + tokens - 1) / tokens - 1 - (tile - begin / tokens - s);
        return end - begin;
    }
    const int s = lane_id();
    const int begin = s < job.n_seqs ? offset(s) : 0, end = s < job.n_seqs ? offset(s + 1) : 0;
    const int rows = max(end - begin, 0), tiles = (rows + tokens - 1) / tokens;
    // Tile number `level` of every sequence that has one, from the highest level down: the lowest level with more than `tile` tiles at and above it.
    if (wave_sum_int(tiles) <= tile) return 0;
    int low = 0, high = (job.n_tokens + tokens - 1) / tokens;  // at and above `low` there are more than `tile`, at and above `high` there are not
    if (high > 64) high = static_cast<int>(wave_max(static_cast<float>(tiles))) + (high > 1 << 24 ? 128 : 0);
    while (high - low > 1) {
        const int middle = (low + high) / 2;
        if (wave_sum_int(max(tiles - middle, 0)) > tile) low = middle;
        else high = middle;
    }
    const int rank = tile - wave_sum_int(max(tiles - low - 1, 0));
    const unsigned long long there = __builtin_amdgcn_ballot_w64(tiles > low);
    const int before = __popcll(there & ((1ull << s) - 1ull));
    const unsigned long long mine = __builtin_amdgcn_ballot_w64(tiles > low && before == rank);
    if (mine == 0ull) return 0;  // (offsets that decrease)
    const int at = __builtin_ctzll(mine);
    first_row = __builtin_amdgcn_readlane(begin, at);
    tile = low;
    return __builtin_amdgcn_readlane(rows, at);
}

// (wavefronts to a SIMD: registers for three where binary16 and heads of 64 need no more, two else)
template <typename T, int kHs, int kR, int kP, int kStepRows>
__global__ __launch_bounds__(64 * kR * kP, sizeof(T) == 2 && kHs == 64 ? 3 : 2) void prompt_kernel(PromptJob job) {
    typedef Shape<kHs, kR, kP, kStepRows> S;
    constexpr bool kLo = sizeof(T) == 4;  // queries have a remainder
    constexpr int kDTiles = kHs / 32, kKSteps = kHs / 16, kStep = S::kStep, kRowBytes = S::kRowBytes, kPieces = S::kPieces;
    constexpr int kTiles = kStep / 32;  // tiles of 32 positions in a step
    extern __shared__ __align__(1024) char lds[];
    const int lane = lane_id(), wave = wave_index();
    const int wr = wave % kR, wp = wave / kR;
    const int r = lane & 31, g = lane >> 5;
    const int tokens_per_wave = 32 / job.shared, tokens = kR * tokens_per_wave;
    // (a KV head's workgroups are n_kv_heads apart: with 8 of them, or a divisor, its rows stay in one die's L2 or few)
    const int kvh = static_cast<int>(blockIdx.x) % job.n_kv_heads;
    int tile = static_cast<int>(blockIdx.x) / job.n_kv_heads, first_row = 0;
    const int rows = find_tile(job, tokens, tile, first_row);
    if (tile < 0 || tile * tokens >= rows) return;
    // positions count from the sequence's first row
    const int first_token = tile * tokens, t0 = first_token + wr * tokens_per_wave;
    const int limit = min(first_token + tokens, rows);                       // the workgroup reads [0, limit)
    const int wave_limit = t0 < rows ? min(t0 + tokens_per_wave, rows) : 0;  // the wavefront attends to [0, wave_limit)
    const int my_tok = t0 + r / job.shared, my_head = r % job.shared;
    const bool valid = my_tok < rows && r < tokens_per_wave * job.shared;
    const int tok_c = min(my_tok, rows - 1);
    const int my_limit = min(tok_c, t0 + tokens_per_wave - 1) + 1;  // this lane's row attends to [0, my_limit)
    const char* kbase = reinterpret_cast<const char*>(job.k + static_cast<size_t>(first_row) * job.kv_stride + kvh * kHs);
    const char* vbase = reinterpret_cast<const char*>(job.v + static_cast<size_t>(first_row) * job.kv_stride + kvh * kHs);
    const size_t row_step = static_cast<size_t>(job.kv_stride) * 2;

    char* stages = lds + wp * S::kStages * S::kStageBytes;
    const unsigned lds_base = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)stages));
    const int steps = (limit + kStep - 1) / kStep, turns = (steps + kP - 1) / kP;
    // Requests of 1 KiB, kRowsPerLoad rows each: a wavefront's are kR apart, so that the order of a row's pieces repeats every kKinds of them,
    // and what a lane adds to a uniform address is the same for those.  Only the last step looks where the rows end (rows behind are the last
    // one again).
    constexpr int kRowsPerLoad = 1024 / kRowBytes, kLoadsPerHalf = S::kHalfBytes / 1024, kEach = kLoadsPerHalf / kR;
    constexpr int kPeriod = kHs == 64 ? 2 : 4, kKinds = kR >= kPeriod ? 1 : kPeriod / kR;
    auto k_order = [](int row) { return kHs == 64 ? (row >> 1) & 7 : row & 15; };
    auto v_order = [](int row) { return kHs == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); };
    const uint32_t row_step32 = static_cast<uint32_t>(row_step);
    uint32_t k_off[kKinds];
#pragma unroll
    for (int i = 0; i < kKinds; ++i) {
        const int row = (wr + kR * i) * kRowsPerLoad + lane / kPieces;
        k_off[i] = lane / kPieces * row_step32 + 16 * ((lane % kPieces) ^ k_order(row));
    }
    const uint32_t v_off = lane / kPieces * row_step32 + 16 * ((lane % kPieces) ^ v_order(lane / kPieces));
    auto load_lds = [](const char* base, uint32_t offset, unsigned at) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1\n" ::"v"(offset), "s"(base), "s"(at) : "memory");
    };
    auto request = [&](int turn) {
        const int p0 = (turn * kP + wp) * kStep;
        if (p0 >= limit) return;  // (one row of wavefronts: never)
        const unsigned at = __builtin_amdgcn_readfirstlane(lds_base + (turn % S::kStages) * S::kStageBytes);
        if (p0 + kStep <= limit) {
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int load = wr + kR * i;
                    const char* base = (w ? vbase : kbase) + static_cast<size_t>(p0 + load * kRowsPerLoad) * row_step;
                    load_lds(base, w ? v_off : k_off[i % kKinds], at + w * S::kHalfBytes + load * 1024);
                }
        } else {
            const char* base[2] = {kbase + static_cast<size_t>(p0) * row_step, vbase + static_cast<size_t>(p0) * row_step};
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int load = wr + kR * i, row = load * kRowsPerLoad + lane / kPieces;
                const uint32_t off = static_cast<uint32_t>(min(row, limit - 1 - p0)) * row_step32;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    load_lds(base[w], off + 16 * ((lane % kPieces) ^ (w ? v_order(row) : k_order(row))), at + w * S::kHalfBytes + load * 1024);
            }
        }
    };
    request(0);

    half8_t qh[kKSteps], ql[kLo ? kKSteps : 1];
    {
        const T* qrow = static_cast<const T*>(job.q) + static_cast<size_t>(first_row + tok_c) * job.q_stride + (kvh * job.shared + my_head) * kHs + 8 * g;
#pragma unroll
        for (int s = 0; s < kKSteps; ++s) {
            if constexpr (kLo) {
                const floatx4 a = as_float4(load16(qrow + 16 * s)), b = as_float4(load16(qrow + 16 * s + 4));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = e < 4 ? a[e & 3] : b[e & 3];
                    const half_t h = static_cast<half_t>(v);
                    qh[s][e] = h;
                    ql[s][e] = static_cast<half_t>(v - static_cast<float>(h));
                }
            } else {
                qh[s] = as_half8(load16(qrow + 16 * s));
            }
        }
    }
    floatx16 o[kDTiles];
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    const float scale = 1.44269504088896341f / sqrtf(static_cast<float>(kHs));
    float top = 0.0f, lsum = 0.0f;  // (the sum over this lane's own positions)
    bool seen = false;              // the row has attended to something: top is a score less kLift
    float minus_one = -1.0f;
    asm("" : "+v"(minus_one));

    // (Q has landed: the loops, whose own requests are under way, do not wait for it)
    if constexpr (!kLo)
#pragma unroll
        for (int s = 0; s < kKSteps; ++s) asm volatile("" : "+v"(qh[s]));

    // where this lane reads its fragments of a tile: K row r, pieces 2 s + g; V rows 4 g + (lane % 16) / 4 of the first
    // sixteen, dimensions 32 dt + 16 (lane / 16 % 2) + 4 (lane % 4) ..
    int k_at[kKSteps], v_at[kDTiles];
#pragma unroll
    for (int s = 0; s < kKSteps; ++s) k_at[s] = r * kRowBytes + 16 * ((2 * s + g) ^ (kHs == 64 ? (r >> 1) & 7 : r & 15));
    {
        const int row = 4 * g + ((lane & 15) >> 2);
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt) {
            const int piece = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            v_at[dt] = row * kRowBytes + 16 * (piece ^ (kHs == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3))) + 8 * (lane & 1);
        }
    }

    // `count` tiles of 32 positions from p0 on, K rows at `keys`, V rows at `values`.  kPartly: some row of the wavefront does not attend to all of
    // them (the last tiles of a walk).
    auto walk = [&](auto partly, auto count, int p0, const char* keys, const char* values) {
        constexpr bool kPartly = decltype(partly)::value;
        constexpr int kTiles = decltype(count)::value;
        floatx16 st[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int e = 0; e < 16; ++e) st[t][e] = 0.0f;
#pragma unroll
            for (int s = 0; s < kKSteps; ++s) {
                const half8_t kf = *reinterpret_cast<const half8_t*>(keys + t * 32 * kRowBytes + k_at[s]);
                st[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[s], st[t], 0, 0, 0);
                if constexpr (kLo) st[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[s], st[t], 0, 0, 0);
            }
        }
        if constexpr (!kPartly) {
            // Six of K's fragments on their way before the first product, another with each product (left to the compiler, each is requested when the
            // last one is used: 2048 rows, 32 heads of 128, binary16, 58 us for 54).
            constexpr int kFragments = kTiles * kKSteps, kAhead = kFragments < 6 ? kFragments : 6, kProducts = kLo ? 2 : 1;
            constexpr int kMatrix = 0x008, kLdsRead = 0x100;
            __builtin_amdgcn_sched_group_barrier(kLdsRead, kAhead, 0);
#pragma unroll
            for (int i = 0; i < kFragments - kAhead; ++i) {
                __builtin_amdgcn_sched_group_barrier(kMatrix, kProducts, 0);
                __builtin_amdgcn_sched_group_barrier(kLdsRead, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(kMatrix, kProducts * kAhead, 0);
        }
        if constexpr (kPartly) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int pos = p0 + 32 * t + 8 * (e >> 2) + 4 * g + (e & 3);
                    st[t][e] = pos < my_limit ? st[t][e] : -INFINITY;
                }
        }
        float step_top = -INFINITY;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) step_top = fmaxf(step_top, st[t][e]);
        step_top = halves_max(step_top) * scale;
        if constexpr (kLo) step_top = __builtin_ceilf(step_top);
        const bool moves = step_top > (seen ? top + (kLift + kSlack) : -INFINITY);
        if (__builtin_amdgcn_ballot_w64(moves) != 0ull) {  // (uniform)
            const float to = moves ? step_top - kLift : top;
            const float corr = __builtin_amdgcn_exp2f(seen ? top - to : 0.0f);  // (nothing to rescale before a row's first step)
            top = to;
            lsum *= corr;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= corr;
            seen = seen || moves;
        }
        auto values_of = [&](int s2, int dt) {
            union {
                short4_t part[2];
                half8_t whole;
            } vf;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                vf.part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4_t*)(values + v_at[dt] + (16 * s2 + 8 * j) * kRowBytes));
            return vf.whole;
        };
        bool odd = false;  // an infinity or NaN among V rows that some row may not attend to
        if constexpr (kPartly) {
            uint32_t any = 0;
#pragma unroll
            for (int s2 = 0; s2 < 2 * kTiles; ++s2)
#pragma unroll
                for (int dt = 0; dt < kDTiles; ++dt) {
                    const uintx4 u = __builtin_bit_cast(uintx4, values_of(s2, dt));
#pragma unroll
                    for (int i = 0; i < 4; ++i) any |= (u[i] & 0x7FFF7FFFu) + 0x04000400u;  // (the exponent's carry)
                }
            odd = __builtin_amdgcn_ballot_w64((any & 0x80008000u) != 0u) != 0ull;
        }
        float step_sum = 0.0f;  // (of its own, so that the running sum is rounded once a step)
#pragma unroll
        for (int s2 = 0; s2 < 2 * kTiles; ++s2) {
            half8_t ph, pl;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float s_0 = st[s2 >> 1][8 * (s2 & 1) + e], s_1 = st[s2 >> 1][8 * (s2 & 1) + e + 1];
                const float p_0 = __builtin_amdgcn_exp2f(fmaf(s_0, scale, -top)), p_1 = __builtin_amdgcn_exp2f(fmaf(s_1, scale, -top));
                // (the packed pair and the factor -1 are hidden from the compiler, which would otherwise round every value a second time to
                // subtract it)
                uint32_t packed = __builtin_bit_cast(uint32_t, half2_t{static_cast<half_t>(p_0), static_cast<half_t>(p_1)});
                asm("" : "+v"(packed));
                const half2_t h = __builtin_bit_cast(half2_t, packed);
                ph[e] = h[0];
                ph[e + 1] = h[1];
                step_sum += p_0 + p_1;
                pl[e] = static_cast<half_t>(fmaf(static_cast<float>(h[0]), minus_one, p_0));
                pl[e + 1] = static_cast<half_t>(fmaf(static_cast<float>(h[1]), minus_one, p_1));
            }
            if (kPartly && odd) {
                // (uniform) A weight of zero would not keep it out.  One token after the other, with the rows behind it cleared; a lane's output is
                // its own token's.
                for (int token = 0; token < tokens_per_wave; ++token) {
                    const int end = t0 + token + 1 - p0 - 16 * s2 - 4 * g;  // positions 0..3 and 8..11 from here are this lane's
#pragma unroll
                    for (int dt = 0; dt < kDTiles; ++dt) {
                        half8_t seen_v = values_of(s2, dt);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if ((e & 3) + 8 * (e >> 2) >= end) seen_v[e] = static_cast<half_t>(0.0f);
                        floatx16 with = __builtin_amdgcn_mfma_f32_32x32x16_f16(seen_v, ph, o[dt], 0, 0, 0);
                        with = __builtin_amdgcn_mfma_f32_32x32x16_f16(seen_v, pl, with, 0, 0, 0);
                        if (my_tok == t0 + token) o[dt] = with;
                    }
                }
            } else {
#pragma unroll
                for (int dt = 0; dt < kDTiles; ++dt) {
                    const half8_t v = values_of(s2, dt);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[dt], 0, 0, 0);
                }
            }
        }
        lsum += step_sum;
    };
    auto rows_of = [&](int turn) -> const char* {  // K rows of a turn's step, V rows behind them; the next ones requested
        // (the step's rows have landed, and nobody reads the stage the next requests go to any more)
        wait_requests<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if constexpr (kR > 1) __syncthreads();
        if (turn + 1 < turns) request(turn + 1);
        return stages + (turn % S::kStages) * S::kStageBytes;
    };
    // First the steps that every row of the wavefront attends to, then those that some do not.  (Two loops: with a branch in one, every step
    // would copy `o` between the registers that its two ways have it in.)
    const int whole_steps = (t0 + 1) / kStep, whole_turns = min(turns, (max(whole_steps - wp, 0) + kP - 1) / kP);
    int turn = 0;
    for (; turn < whole_turns; ++turn) {
        const char* keys = rows_of(turn);
        walk(std::false_type{}, std::integral_constant<int, kTiles>{}, (turn * kP + wp) * kStep, keys, keys + S::kHalfBytes);
    }
    for (; turn < turns; ++turn) {
        const char* keys = rows_of(turn);
        const int p0 = (turn * kP + wp) * kStep;
#pragma unroll 1
        for (int t = 0; t < kTiles && p0 + 32 * t < wave_limit; ++t)
            walk(std::true_type{}, std::integral_constant<int, 1>{}, p0 + 32 * t, keys + t * 32 * kRowBytes, keys + S::kHalfBytes + t * 32 * kRowBytes);
    }
    lsum = halves_sum(lsum);
    T* out_row = static_cast<T*>(job.out) + static_cast<size_t>(first_row + tok_c) * job.out_stride + (kvh * job.shared + my_head) * kHs + 4 * g;
    auto store4 = [&](int four, floatx4 v) {
        const int at = 32 * (four >> 2) + 8 * (four & 3);
        if constexpr (kLo) {
            *reinterpret_cast<floatx4*>(out_row + at) = v;
        } else {
            half4_t h;
#pragma unroll
            for (int u = 0; u < 4; ++u) h[u] = static_cast<half_t>(v[u]);
            *reinterpret_cast<half4_t*>(out_row + at) = h;
        }
    };
    constexpr int kFours = kHs / 8;
    auto four_of = [&](int four) {
        const floatx16& of = o[four >> 2];
        const int at = 4 * (four & 3);
        return floatx4{of[at], of[at + 1], of[at + 2], of[at + 3]};
    };
    if constexpr (kP == 1) {
        if (!valid) return;
        const float inv_sum = 1.0f / lsum;
#pragma unroll
        for (int four = 0; four < kFours; ++four) store4(four, four_of(four) * inv_sum);
    } else {
        // The wavefronts of a row meet in LDS, lane for lane: each leaves its (maximum, sum, output), and each adds up its share of the
        // output's pieces of four values in the order of the wavefronts.  Those past the last step have left nothing and are not read.
        if (!seen) top = -INFINITY;
        __syncthreads();  // (the stages are free)
        constexpr int kPart = S::kPartFloats;
        const int parts = min(steps, kP);
        float* merge = reinterpret_cast<float*>(lds) + wr * kP * kPart;
        if (wp < parts) {
            float* mine = merge + wp * kPart;
            mine[lane] = top;
            mine[64 + lane] = lsum;
#pragma unroll
            for (int four = 0; four < kFours; ++four) *reinterpret_cast<floatx4*>(mine + 128 + 256 * four + 4 * lane) = four_of(four);
        }
        __syncthreads();
        if (!valid) return;
        float weight[kP], all_top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kP; ++w) {
            weight[w] = w < parts ? merge[w * kPart + lane] : -INFINITY;
            all_top = fmaxf(all_top, weight[w]);
        }
        if (all_top == -INFINITY) all_top = 0.0f;  // (no score was a number)
#pragma unroll
        for (int w = 0; w < kP; ++w) {
            weight[w] = __builtin_amdgcn_exp2f(weight[w] - all_top);
            if (w < parts) total = fmaf(merge[w * kPart + 64 + lane], weight[w], total);
        }
        const float inv_sum = 1.0f / total;
#pragma unroll
        for (int f = 0; f < kFours / kP; ++f) {
            const int four = wp + kP * f;
            floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kP; ++w) {
                if (w >= parts) break;
                const floatx4 a = *reinterpret_cast<const floatx4*>(merge + w * kPart + 128 + 256 * four + 4 * lane);
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = fmaf(a[u], weight[w], v[u]);
            }
            store4(four, v * inv_sum);
        }
    }
}

template <typename T, int kHs, int kR, int kP, int kStepRows>
lpp_status launch_as(const PromptJob& job, int n_seqs) {
    constexpr int kLds = Shape<kHs, kR, kP, kStepRows>::kLdsBytes;
    const auto kernel = &prompt_kernel<T, kHs, kR, kP, kStepRows>;
    if constexpr (kLds > 64 * 1024) {
        static bool sized[64] = {};
        LPP_TRY(tell_lds(reinterpret_cast<const void*>(kernel), kLds, sized));
    }
    // (as many tile numbers as find_tile gives to sequences of any lengths: one more than whole tiles for each sequence, and up to kWave of them only
    // for those that have rows.  A number without a tile costs a workgroup that finds out: one prompt of 300 rows, 32 heads of 64 on 8, fp32, among 300
    // sequences 10.3 us, among 5000 100, by itself 8.3.)
    const int tokens = kR * (32 / job.shared);
    const long long tiles = job.n_tokens / tokens + (n_seqs <= dev::kWave && n_seqs > job.n_tokens ? job.n_tokens : n_seqs);
    const long long blocks = tiles * job.n_kv_heads;
    LPP_REQUIRE(blocks * 64 * kR * kP < (1ll << 32), "lpp_prompt_attention: %d rows of %d sequences and %d KV heads are too many for a launch", job.n_tokens,
                n_seqs, job.n_kv_heads);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * kR * kP), kLds, stream(), job);
    LPP_CHECK_LAUNCH("prompt_kernel");
    return LPP_OK;
}

// Which shape: the fewer tiles of 32 rows there are for each compute unit, the more wavefronts share a walk.  us, one prompt, 1 x 4 / 2 x 2 / 4 x 1,
// 32 heads of 64 on 8, fp32: 256 rows (one tile a compute unit) 6.4 / 7.9 / 10.3; 512 9.2 / 11.4 / 14.3; 700 16.0 / 14.3 / 16.6; 1024 21.1 / 19.8 /
// 22.9; 1500 36.7 / 34.5 / 32.4; 2048 58 / 53 / 48; 6000 364 / 327 / 284.  32 heads of 128, binary16: 256 7.5 / 8.9 / 11.6; 400 13.2 / 11.8 / 14.7;
// 1024 35 / 23 / 28.5; 1500 61 / 41 / 42; 2048 100 / 64 / 63; 6000 640 / 447 / 401; of 64: 512 7.4 / 9.2 / 11.8; 700 12.6 / 11.1 / 14.7; 1500 28 / 25 /
// 27; 2048 45.5 / 39.2 / 38.6.  Steps of 4 x 1: 128 positions (fp32, heads of 64; 64: 302 us at 6000 rows for 292), 64 (binary16, heads of 128; 32: 410
// for 401; heads of 64, where three workgroups fit on a compute unit so: 7 prompts of up to 1500 rows 53.6 us, 60 with 128) or 32 (fp32, heads of 128,
// where 64 spill: the same prompts 122 us for 131).  (Built when binary16 weights had no remainder, 321 us at 6000 rows, and no faster: 8 x 1, 326
// and 331; the products of the next step formed between this one's weights, this step's products and weights in turn, a third stage, other
// priorities for the products.)
template <typename T, int kHs>
lpp_status launch(const PromptJob& job, int n_seqs) {
    const long long tiles = (static_cast<long long>(job.n_tokens) * job.shared + 31) / 32 * job.n_kv_heads;  // of 32 rows
    if (tiles <= (kHs == 64 ? 2ll : 1ll) * compute_units()) return launch_as<T, kHs, 1, 4, 32>(job, n_seqs);
    if (tiles <= 6ll * compute_units()) return launch_as<T, kHs, 2, 2, 32>(job, n_seqs);
    return launch_as<T, kHs, 4, 1, sizeof(T) == 2 ? 64 : kHs == 64 ? 128 : 32>(job, n_seqs);
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
    LPP_REQUIRE(kv_stride <= 1 << 24, "lpp_prompt_attention: kv_stride = %d is beyond 2^24", kv_stride);
    if (n_tokens == 0) return LPP_OK;
    LPP_REQUIRE(d_out && d_q && d_k && d_v, "lpp_prompt_attention: null pointer");
    const int size = type == LPP_F32 ? 4 : 2, per16 = 16 / size;
    const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    LPP_REQUIRE(aligned(d_out) && aligned(d_q) && aligned(d_k) && aligned(d_v) && q_stride % per16 == 0 && out_stride % per16 == 0 && kv_stride % 8 == 0,
                "lpp_prompt_attention: rows must start at multiples of 16 bytes");
    const auto bytes = [&](int stride, long long row, int of) { return (static_cast<size_t>(n_tokens - 1) * stride + row) * of; };
    const size_t out_bytes = bytes(out_stride, width, size), q_bytes = bytes(q_stride, width, size), kv_bytes = bytes(kv_stride, kv_width, 2);
    LPP_REQUIRE(!ranges_overlap(d_out, out_bytes, d_q, q_bytes) && !ranges_overlap(d_out, out_bytes, d_k, kv_bytes) &&
                    !ranges_overlap(d_out, out_bytes, d_v, kv_bytes) &&
                    (d_offsets == nullptr || !ranges_overlap(d_out, out_bytes, d_offsets, (static_cast<size_t>(n_seqs) + 1) * 4)),
                "lpp_prompt_attention: d_out overlaps an input");
    PromptJob job;
    job.out = d_out;
    job.q = d_q;
    job.k = reinterpret_cast<const dev::half_t*>(d_k);
    job.v = reinterpret_cast<const dev::half_t*>(d_v);
    job.offsets = d_offsets;
    job.n_seqs = n_seqs;
    job.n_tokens = n_tokens;
    job.shared = n_heads / n_kv_heads;
    job.n_kv_heads = n_kv_heads;
    job.q_stride = q_stride;
    job.kv_stride = kv_stride;
    job.out_stride = out_stride;
    if (type == LPP_F32) return head_size == 64 ? launch<float, 64>(job, n_seqs) : launch<float, 128>(job, n_seqs);
    return head_size == 64 ? launch<dev::half_t, 64>(job, n_seqs) : launch<dev::half_t, 128>(job, n_seqs);
}

}  // extern "C"
