// ops_kv4_attention.hip -- lpp_kv4_attention, lpp_kv4_attention_workspace:
// attention of a few new rows over the cache of 4 bits, and the weight each
// position got.
#include "kv4.hpp"

namespace lpp {
namespace {

using namespace dev;

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;       // of a tile: (16 / shared) new rows x the query heads of a KV head
constexpr int kStep = 32;       // positions a wavefront takes at a time
constexpr int kWaves = 4, kThreads = kWave * kWaves;
constexpr int kMaxSplits = 64;  // ranges that a sequence's positions are cut into
constexpr float kSlack = 6.0f;

struct AttendJob {
    float* out;
    const float* q;
    Kv4Layer cache;
    const int* starts;
    float* mass;
    float2* stats;     // [sequence][KV head][tile][range][16]: maximum (in powers of two) and sum of a range
    float* partials;   // [sequence][KV head][tile][range][16][head_size]
    int n_q, n_kv_heads, shared, seq_len, splits, least, tiles;
};

__device__ __forceinline__ int rows_end(int start, int row, int seq_len) {
    return static_cast<int>(min(max(static_cast<long long>(start) + row + 1, 0ll), static_cast<long long>(seq_len)));
}
// How many positions a range has: whole steps of a workgroup, `least` at least.
__device__ __forceinline__ int range_of(int positions, int splits, int least) {
    constexpr int kWhole = kStep * kWaves;
    const int even = (positions + splits - 1) / splits;
    return max(least, (even + kWhole - 1) / kWhole * kWhole);
}

__device__ __forceinline__ float rows_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned m = __float_as_uint(fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1])));
    const auto halves = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}
// A lane's part of 16 rows of codes: of position lane % 16, the kHs / 4 values from kHs / 4 * (lane / 16) on.
template <int kHs>
struct Piece {
    static constexpr int kWords = kHs / 32;
    uint32_t codes[kWords], pair;
    __device__ __forceinline__ void load(const uint32_t* codes_of_head, const uint32_t* scales_of_head, int pos, int part) {
        const uint32_t* from = codes_of_head + static_cast<size_t>(pos) * (kHs / 8) + part * kWords;
        if constexpr (kWords == 4) {
            const uintx4 all = load16(from);
#pragma unroll
            for (int i = 0; i < 4; ++i) codes[i] = all[i];
        } else {
            const uint2 all = *reinterpret_cast<const uint2*>(from);
            codes[0] = all.x;
            codes[1] = all.y;
        }
        pair = scales_of_head[static_cast<size_t>(pos) * (kHs / kKv4Group) + part * kWords / 4];
    }
    __device__ __forceinline__ half8_t values(int i) const { return kv4_values(codes[i], pair); }
    // Whether a value may be infinite or NaN.
    __device__ __forceinline__ bool may_be_nonfinite() const {
        const half2_t both = __builtin_bit_cast(half2_t, pair);
        return !(fmaf(15.0f, fabsf(static_cast<float>(both[0])), fabsf(static_cast<float>(both[1]))) < 65504.0f);
    }
};

// Q of a tile as B operands: column lane % 16, the values that a K piece's words have; heads and remainders.
template <int kHs>
struct Queries {
    static constexpr int kWords = kHs / 32;
    half8_t high[kWords], low[kWords];
    __device__ __forceinline__ void load(const float* row, int part) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const float* from = row + part * kWords * 8 + 8 * i;
            const floatx4 a = as_float4(load16(from)), b = as_float4(load16(from + 4));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = e < 4 ? a[e & 3] : b[e & 3];
                high[i][e] = static_cast<half_t>(v);
                low[i][e] = static_cast<half_t>(v - static_cast<float>(high[i][e]));
            }
        }
    }
    // scores of 16 positions: lane: column lane % 16, positions 4 (lane / 16) ..
    __device__ __forceinline__ floatx4 scores(const Piece<kHs>& k) const {
        floatx4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const half8_t kv = k.values(i);
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, high[i], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, low[i], s, 0, 0, 0);
        }
        return s;
    }
};

// Which row a column of a tile is.
struct Column {
    int token, head;
    bool valid;
    __device__ __forceinline__ Column(const AttendJob& job, int tile, int column) {
        const int tokens = kRows / job.shared;
        token = tile * tokens + column / job.shared;
        head = column % job.shared;
        valid = column < tokens * job.shared && token < job.n_q;
        token = min(token, min(tile * tokens + tokens, job.n_q) - 1);
    }
    __device__ __forceinline__ size_t at(const AttendJob& job, int s, int kvh) const {
        return (static_cast<size_t>(s) * job.n_q + token) * job.n_kv_heads * job.shared + kvh * job.shared + head;
    }
};

template <int kHs>
__global__ __launch_bounds__(kThreads) void attend_kernel(AttendJob job) {
    constexpr int kDTiles = kHs / 16, kWords = kHs / 32, kRowBytes = 2 * kHs;
    constexpr int kPad = kHs + 4, kPart = kRows * kPad + 2 * kRows;  // floats a wavefront leaves for the merge
    constexpr int kWaveBytes = kPart * 4;
    static_assert(kWaveBytes >= kStep * kRowBytes, "V rows of a step");
    __shared__ __align__(16) char lds[kWaves * kWaveBytes];
    const int lane = lane_id(), wave = wave_index(), column = lane & 15, part = lane >> 4;
    const int split = static_cast<int>(blockIdx.x) % job.splits, tile = static_cast<int>(blockIdx.x) / job.splits, kvh = blockIdx.y, s = blockIdx.z;
    const int tokens = kRows / job.shared, start = job.starts[s];
    const int all_end = rows_end(start, job.n_q - 1, job.seq_len);
    const int range = range_of(all_end, job.splits, job.least);
    const int begin = split * range;
    if (begin >= all_end && split > 0) return;
    const int tile_end = rows_end(start, min(tile * tokens + tokens, job.n_q) - 1, job.seq_len);
    const int end = min(begin + range, tile_end);  // (at or before `begin`: the tile's rows attend to nothing here)
    const bool only = range >= all_end;            // (uniform over the sequence: no merge)
    const Column mine(job, tile, column);
    const int my_end = rows_end(start, mine.token, job.seq_len), first_end = rows_end(start, tile * tokens, job.seq_len);
    const size_t head_rows = (static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.seq_len;
    const uint32_t* codes[2];
    const uint32_t* scales[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        codes[w] = job.cache.codes[w] + head_rows * (kHs / 8);
        scales[w] = job.cache.scales[w] + head_rows * (kHs / kKv4Group);
    }
    Queries<kHs> q;
    q.load(job.q + mine.at(job, s, kvh) * kHs, part);

    floatx4 o[kDTiles];
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) o[dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const float scale = 1.44269504088896341f / sqrtf(static_cast<float>(kHs));
    float top = 0.0f, lsum = 0.0f;  // (the sum over this lane's own positions)
    bool seen = false;              // the row has attended to something: top is a score
    float minus_one = -1.0f;
    asm("" : "+v"(minus_one));

    // V rows of a step, in this wavefront's own LDS: 16-byte pieces in an order that keeps writes and transposing reads free of bank
    // conflicts
    char* values = lds + wave * kWaveBytes;
    auto swizzle = [](int row) { return kHs == 64 ? 2 * ((row >> 1) & 3) : 4 * (row & 3) + ((row >> 2) & 3); };
    int v_at[kDTiles];
    {
        const int row = 4 * part + ((lane & 15) >> 2);
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt) v_at[dt] = row * kRowBytes + 16 * ((2 * dt + ((lane & 3) >> 1)) ^ swizzle(row)) + 8 * (lane & 1);
    }

    Piece<kHs> next[2][2];  // [K, V][first, second sixteen positions]
    auto request = [&](int p0) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < 2; ++w) next[w][t].load(codes[w], scales[w], min(p0 + 16 * t + column, end - 1), part);
    };
    const int first = begin + wave * kStep;
    if (first < end) request(first);
    for (int p0 = first; p0 < end; p0 += kStep * kWaves) {
        Piece<kHs> now[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < 2; ++w) now[w][t] = next[w][t];
        if (p0 + kStep * kWaves < end) request(p0 + kStep * kWaves);
        const bool partly = p0 + kStep > first_end;  // (uniform) some row does not attend to the whole step
        floatx4 st[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) st[t] = q.scores(now[0][t]);
        // V into LDS.  Rows behind the tile's last position are cleared: a weight of zero does not keep an infinity or NaN out.
        bool odd = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int row = 16 * t + column;
            const bool live = p0 + row < tile_end;
            odd = odd || (live && now[1][t].may_be_nonfinite());
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                half8_t v = now[1][t].values(i);
                if (partly && !live) v = half8_t{};
                *reinterpret_cast<half8_t*>(values + row * kRowBytes + 16 * ((kWords * part + i) ^ swizzle(row))) = v;
            }
        }
        odd = __builtin_amdgcn_ballot_w64(odd) != 0ull;
        if (partly) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) st[t][e] = p0 + 16 * t + 4 * part + e < my_end ? st[t][e] : -INFINITY;
        }
        float step_top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) step_top = fmaxf(step_top, st[t][e]);
        step_top = __builtin_ceilf(rows_max(step_top) * scale);
        const bool moves = step_top > (seen ? top + kSlack : -INFINITY);
        if (__builtin_amdgcn_ballot_w64(moves) != 0ull) {  // (uniform)
            const float to = moves ? step_top : top;
            const float corr = __builtin_amdgcn_exp2f(seen ? top - to : 0.0f);  // (nothing to rescale before a row's first step)
            top = to;
            lsum *= corr;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) o[dt] *= corr;
            seen = seen || moves;
        }
        half8_t ph, pl;
        float step_sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float p_0 = __builtin_amdgcn_exp2f(fmaf(st[e >> 2][e & 3], scale, -top)), p_1 = __builtin_amdgcn_exp2f(fmaf(st[e >> 2][(e & 3) + 1], scale, -top));
            step_sum += p_0 + p_1;
            // (hidden from the compiler, which would otherwise round every value a second time to subtract it)
            uint32_t packed = __builtin_bit_cast(uint32_t, half2_t{static_cast<half_t>(p_0), static_cast<half_t>(p_1)});
            asm("" : "+v"(packed));
            const half2_t h = __builtin_bit_cast(half2_t, packed);
            ph[e] = h[0];
            ph[e + 1] = h[1];
            pl[e] = static_cast<half_t>(fmaf(static_cast<float>(h[0]), minus_one, p_0));
            pl[e + 1] = static_cast<half_t>(fmaf(static_cast<float>(h[1]), minus_one, p_1));
        }
        lsum += step_sum;
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt) {
            union {
                short4_t half[2];
                half8_t whole;
            } vf;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                vf.half[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(values + v_at[dt] + 16 * t * kRowBytes));
            if (odd) {
                // (uniform) An infinity or NaN, perhaps, among the step's V rows: one token after the other, with the rows behind it cleared; a
                // lane's output is its own token's.  The weights' remainders, of either sign, meet the finite values only.
                for (int token = 0; token < tokens; ++token) {
                    const int token_end = rows_end(start, tile * tokens + token, job.seq_len) - p0 - 4 * part;
                    half8_t v = vf.whole;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((e & 3) + 16 * (e >> 2) >= token_end) v[e] = static_cast<half_t>(0.0f);
                    floatx4 with = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[dt], 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (!(fabsf(static_cast<float>(v[e])) < INFINITY)) v[e] = static_cast<half_t>(0.0f);
                    with = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, with, 0, 0, 0);
                    if (column / job.shared == token) o[dt] = with;
                }
            } else {
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf.whole, ph, o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf.whole, pl, o[dt], 0, 0, 0);
            }
        }
    }
    lsum = rows_sum(lsum);
    if (!seen) top = -INFINITY;

    // The wavefronts meet in LDS, each thread adding four values of a row in the order of the wavefronts.
    float* all = reinterpret_cast<float*>(lds);
    float* my_part = all + wave * kPart;
    // (its own V rows are read: the values are in registers)
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) *reinterpret_cast<floatx4*>(my_part + column * kPad + 16 * dt + 4 * part) = o[dt];
    if (part == 0) {
        my_part[kRows * kPad + column] = top;
        my_part[kRows * kPad + kRows + column] = lsum;
    }
    __syncthreads();
    const size_t slot = ((static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.tiles + tile) * job.splits + split;
    constexpr int kFours = kHs / 4;
    for (int i = threadIdx.x; i < kRows * kFours; i += kThreads) {
        const int row = i / kFours, four = i % kFours;
        const Column its(job, tile, row);
        if (!its.valid) continue;
        float weight[kWaves], all_top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            weight[w] = all[w * kPart + kRows * kPad + row];
            all_top = fmaxf(all_top, weight[w]);
        }
        const float reference = all_top == -INFINITY ? 0.0f : all_top;  // (nothing seen, or no score was a number)
        floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            weight[w] = __builtin_amdgcn_exp2f(weight[w] - reference);
            total = fmaf(all[w * kPart + kRows * kPad + kRows + row], weight[w], total);
            const floatx4 a = *reinterpret_cast<const floatx4*>(all + w * kPart + row * kPad + 4 * four);
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = fmaf(a[u], weight[w], v[u]);
        }
        if (only) {
            const bool any = rows_end(start, its.token, job.seq_len) > 0;
            const float inverse = 1.0f / total;
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = any ? v[u] * inverse : 0.0f;
            *reinterpret_cast<floatx4*>(job.out + its.at(job, s, kvh) * kHs + 4 * four) = v;
        } else {
            *reinterpret_cast<floatx4*>(job.partials + (slot * kRows + row) * kHs + 4 * four) = v;
        }
        if (four == 0) job.stats[slot * kRows + row] = make_float2(all_top, total);
    }
}

// What is left once every range has been walked: blocks before job.tiles (where there are ranges to merge) merge a tile's rows, the others add up
// the weights of kMassPositions positions each.
constexpr int kMassPositions = 2 * kStep * kWaves;

template <int kHs>
__global__ __launch_bounds__(kThreads) void finish_kernel(AttendJob job, int merges) {
    __shared__ float weights[kRows][kMaxSplits];
    __shared__ float tops[kRows], inverses[kRows];
    const int lane = lane_id(), wave = wave_index(), column = lane & 15, part = lane >> 4;
    const int kvh = blockIdx.y, s = blockIdx.z, start = job.starts[s], tokens = kRows / job.shared;
    const int all_end = rows_end(start, job.n_q - 1, job.seq_len);
    const int range = range_of(all_end, job.splits, job.least), active = max((all_end + range - 1) / range, 1);
    const bool merging = static_cast<int>(blockIdx.x) < merges;
    if (merging && active == 1) return;
    const int p_first = (static_cast<int>(blockIdx.x) - merges) * kMassPositions;
    if (!merging && p_first >= all_end) return;

    // (maximum, 1 / sum) of a tile's rows, and every range's weight in them; 16 threads to a row
    auto combine = [&](int tile) {
        const size_t slot = ((static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.tiles + tile) * job.splits;
        const int row = threadIdx.x / 16, at = threadIdx.x % 16;
        const bool live = Column(job, tile, row).valid;
        float2 st[kMaxSplits / 16];
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxSplits / 16; ++i) {
            st[i] = live && at + 16 * i < active ? job.stats[(slot + at + 16 * i) * kRows + row] : make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, st[i].x);
        }
        top = fmaxf(top, dpp_move<kDppXor1>(top));
        top = fmaxf(top, dpp_move<kDppXor2>(top));
        top = fmaxf(top, dpp_move<kDppHalfMirror>(top));
        top = fmaxf(top, dpp_move<kDppMirror>(top));
        if (top == -INFINITY) top = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxSplits / 16; ++i) {
            const float w = __builtin_amdgcn_exp2f(st[i].x - top);
            // (a range that the row does not attend to has left no output)
            weights[row][at + 16 * i] = st[i].x == -INFINITY && st[i].y == 0.0f ? -1.0f : w;
            total = fmaf(st[i].y, w, total);
        }
        total = row16_sum(total);
        if (at == 0) {
            tops[row] = top;
            inverses[row] = live ? 1.0f / total : 0.0f;
        }
    };
    if (merging) {
        const int tile = blockIdx.x;
        combine(tile);
        __syncthreads();
        const size_t slot = ((static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.tiles + tile) * job.splits;
        constexpr int kFours = kHs / 4;
        for (int i = threadIdx.x; i < kRows * kFours; i += kThreads) {
            const int row = i / kFours, four = i % kFours;
            const Column its(job, tile, row);
            if (!its.valid) continue;
            floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
            const float* from = job.partials + (slot * kRows + row) * kHs + 4 * four;
#pragma unroll 8
            for (int k = 0; k < active; ++k) {
                const float w = weights[row][k];
                if (w < 0.0f) continue;
                const floatx4 a = *reinterpret_cast<const floatx4*>(from + static_cast<size_t>(k) * kRows * kHs);
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = fmaf(a[u], w, v[u]);
            }
            const bool any = rows_end(start, its.token, job.seq_len) > 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = any ? v[u] * inverses[row] : 0.0f;
            *reinterpret_cast<floatx4*>(job.out + its.at(job, s, kvh) * kHs + 4 * four) = v;
        }
        return;
    }
    const size_t head_rows = (static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.seq_len;
    const uint32_t* codes = job.cache.codes[0] + head_rows * (kHs / 8);
    const uint32_t* scales = job.cache.scales[0] + head_rows * (kHs / kKv4Group);
    const float scale = 1.44269504088896341f / sqrtf(static_cast<float>(kHs));
    constexpr int kPieces = kMassPositions / (kWaves * 16);
    Piece<kHs> k[kPieces];
    floatx4 sum[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        k[i].load(codes, scales, min(p_first + 16 * (wave + kWaves * i) + column, all_end - 1), part);
        sum[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int tile = 0; tile < job.tiles; ++tile) {
        if (rows_end(start, min(tile * tokens + tokens, job.n_q) - 1, job.seq_len) <= p_first) continue;  // (uniform)
        const Column mine(job, tile, column);
        const int my_end = rows_end(start, mine.token, job.seq_len);
        Queries<kHs> q;
        q.load(job.q + mine.at(job, s, kvh) * kHs, part);
        __syncthreads();
        combine(tile);
        __syncthreads();
        const float top = tops[column], inverse = inverses[column];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p0 = p_first + 16 * (wave + kWaves * i) + 4 * part;
            const floatx4 st = q.scores(k[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = __builtin_amdgcn_exp2f(fmaf(st[e], scale, -top)) * inverse;
                sum[i][e] += row16_sum(mine.valid && p0 + e < my_end ? w : 0.0f);
            }
        }
    }
    float* mass = job.mass + head_rows;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int p0 = p_first + 16 * (wave + kWaves * i) + 4 * part;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (column == e && p0 + e < all_end) mass[p0 + e] += sum[i][e];
    }
}

int tiles_of(int n_q, int shared) { return (n_q + kRows / shared - 1) / (kRows / shared); }

// Ranges a sequence's positions are cut into, and the least positions of one.
struct Split {
    int splits, least;
};
Split split_of(const lpp_kv4_shape& shape, int tiles) {
    const long long heads = static_cast<long long>(shape.n_seqs) * shape.n_kv_heads * tiles;
    Split s;
    s.least = heads >= 2ll * compute_units() ? 1024 : heads * 4 >= compute_units() ? 512 : 256;
    const int most = (shape.seq_len + s.least - 1) / s.least;
    s.splits = most < kMaxSplits ? most : kMaxSplits;
    return s;
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
    const int tiles = tiles_of(n_q, n_heads / shape->n_kv_heads);
    const size_t slots = static_cast<size_t>(shape->n_seqs) * shape->n_kv_heads * tiles * split_of(*shape, tiles).splits;
    *bytes = slots * kRows * (sizeof(float2) + shape->head_size * sizeof(float));
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
    AttendJob job;
    job.out = d_out;
    job.q = d_q;
    job.cache = kv4_layer(d_cache, *shape, layer);
    job.starts = d_starts;
    job.mass = d_mass != nullptr ? d_mass + kv4_layer_rows(*shape) * layer : nullptr;
    job.n_q = n_q;
    job.n_kv_heads = shape->n_kv_heads;
    job.shared = n_heads / shape->n_kv_heads;
    job.seq_len = shape->seq_len;
    job.tiles = tiles_of(n_q, job.shared);
    const Split split = split_of(*shape, job.tiles);
    job.splits = split.splits;
    job.least = split.least;
    const size_t slots = static_cast<size_t>(shape->n_seqs) * shape->n_kv_heads * job.tiles * job.splits;
    job.stats = static_cast<float2*>(d_workspace);
    job.partials = reinterpret_cast<float*>(job.stats + slots * kRows);
    const dim3 grid(static_cast<unsigned>(job.splits) * job.tiles, shape->n_kv_heads, shape->n_seqs);
    if (shape->head_size == 64)
        hipLaunchKernelGGL(attend_kernel<64>, grid, dim3(kThreads), 0, stream(), job);
    else
        hipLaunchKernelGGL(attend_kernel<128>, grid, dim3(kThreads), 0, stream(), job);
    LPP_CHECK_LAUNCH("attend_kernel");
    const int merges = job.splits > 1 ? job.tiles : 0;
    const int blocks = merges + (d_mass != nullptr ? (shape->seq_len + kMassPositions - 1) / kMassPositions : 0);
    if (blocks > 0) {
        const dim3 rest(blocks, shape->n_kv_heads, shape->n_seqs);
        if (shape->head_size == 64)
            hipLaunchKernelGGL(finish_kernel<64>, rest, dim3(kThreads), 0, stream(), job, merges);
        else
            hipLaunchKernelGGL(finish_kernel<128>, rest, dim3(kThreads), 0, stream(), job, merges);
        LPP_CHECK_LAUNCH("finish_kernel");
    }
    return LPP_OK;
}

}  // extern "C"
