// ops_kv4_attention.hip -- lpp_kv4_attention, lpp_kv4_attention_workspace:
// attention of a few new rows over the cache of 4 bits, and the weight each position got.
//
// The sums are those of a softmax in one walk: w(t, p) = 2^(scale q[t] . k[p] - top(t)), with `top` kLift below a score of the row so far, moved
// (and sum and output rescaled) when a score passes that one by more than kSlack.  The positions of a sequence are cut into shares, which leave (top, sum, output) each;
// a second kernel weighs those by 2^(top - largest top) and adds them up in their order.  The weight that a position got needs the row's final
// maximum and sum, so it is the second kernel's too.
//
// What there is to read is 5 bits a value, K and V once for all the query heads of a KV head: 13 instructions make eight binary16 values of a word of
// codes (dev::Kv4Reader), and the matrix cores take 16 rows x 16 positions at a time, the few rows there are beside unused ones, for which nothing
// else would have to be formed.  Queries and weights enter as binary16 head and remainder.  V goes through LDS, for transposing reads.
//
// What bounds it: 32 sequences of up to 8000 positions, 32 heads of 128 on 8: 60 us with the scores kept for the account (3.4 TB/s of the 160 bytes a
// position and KV head; reading alone takes 47), and 9 for it and the merge; the rest is instructions for the codes.  One sequence of 16001, heads of
// 64: 7.6 + 3 us, one of 500: 6.5 us: the time of requests one after the other, a start and a merge.
#include "kv4.hpp"

namespace lpp {
namespace {

using namespace dev;

typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;       // of a tile: (16 / shared) new rows x the query heads of a KV head
constexpr int kStep = 32;       // positions a wavefront takes at a time
constexpr int kMaxSplits = 64;  // shares that a sequence's positions are cut into

struct AttendJob {
    float* out;
    const float* q;
    Kv4Layer cache;
    const int* starts;
    float* mass;
    float2* stats;     // [sequence][KV head][tile][share][rows]: maximum (in powers of two) and sum of a share
    float* partials;   // [sequence][KV head][tile][share][rows][head_size]
    float* scores;     // for the account: [sequence][KV head][step][rows][kStep]; null if there is none, or it is made from K again
    int rows, steps;  // of a tile; that seq_len has
    unsigned heads;  // n_seqs times n_kv_heads
    int n_seqs, n_q, n_kv_heads, shared, seq_len, splits, least, tiles;
    float per_workgroup;  // KV heads times tiles over the shares there should be
    unsigned per_shared;  // 65536 / shared, rounded up: column * per_shared >> 16 is column / shared for columns below 16
    // (a start outside -n_q .. seq_len says no more than the ends of that)
    __device__ __forceinline__ int start_of(int s) const { return min(max(starts[s], -n_q), seq_len); }
    __device__ __forceinline__ int end_of(int start, int row) const { return min(max(start + row + 1, 0), seq_len); }
    __device__ __forceinline__ int tokens() const { return static_cast<int>(kRows * per_shared >> 16); }  // of a tile
    // How many shares a sequence's `positions` are cut into: of all sequences' positions, as many to each as gives `workgroups` of them in all,
    // but no fewer than `least`.  (All lanes call it and read the sequences' starts, 64 at a time; the same sum in every workgroup.  Of more than
    // 256 sequences all are taken to be as long as this one, which leaves one that is much longer than the others too few shares: with 300, one of 30000
    // positions and the others of 30, 8 KV heads of 64, 176 us for 75 with the sum.  Any others pay for the sum: 300 of 30 positions 33 us for 22, of 1000
    // 64 for 52; 1000 of up to 2000 238 for 158; 4000 1129 for 555.)
    __device__ __forceinline__ int shares_of(int positions) const {
        float all = n_seqs > 4 * kWave ? static_cast<float>(positions) * n_seqs : 0.0f;
        if (n_seqs <= 4 * kWave)
            for (int s0 = 0; s0 < n_seqs; s0 += kWave) {
                const int s = s0 + lane_id();
                all += wave_sum(s < n_seqs ? static_cast<float>(end_of(start_of(s), n_q - 1)) : 0.0f);
            }
        const int each = max(least, static_cast<int>(fminf(all * per_workgroup, 1e9f)));
        return max(min((positions + each - 1) / each, splits), 1);
    }
};

__device__ __forceinline__ float rows_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned m = __float_as_uint(fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1])));
    const auto halves = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}
// A lane's part of 16 rows of codes: of position lane % 16, the kHs / 4 values from kHs / 4 * (lane / 16) on, and their scale and lowest
// value.
template <int kHs>
struct Piece {
    static constexpr int kWords = kHs / 32;
    uint32_t codes[kWords], pair;
    // (a head's rows are within 2^31 bytes: a uniform base and an offset of 32 bits)
    __device__ __forceinline__ void load(const uint32_t* codes_of_head, int pos, int part) {
        const char* from = reinterpret_cast<const char*>(codes_of_head) + (static_cast<uint32_t>(pos) * (kHs / 2) + static_cast<uint32_t>(part) * (kWords * 4));
        typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
        const Words all = __builtin_nontemporal_load(reinterpret_cast<const Words*>(from));
#pragma unroll
        for (int i = 0; i < kWords; ++i) codes[i] = all[i];
    }
    __device__ __forceinline__ half8_t values(const Kv4Reader& read, int i) const { return read(codes[i], pair); }
    // Whether a value may be infinite or NaN.
    __device__ __forceinline__ bool may_be_nonfinite() const {
        const half2_t both = __builtin_bit_cast(half2_t, pair);
        return !(fmaf(15.0f, fabsf(static_cast<float>(both[0])), fabsf(static_cast<float>(both[1]))) < 65504.0f);
    }
};

// The scales of 64 rows (32 of K and 32 of V, or 64 of K): a lane requests a row's and a wavefront all of them at once; through its own LDS they get
// to the lanes that have the codes.  (Requested by those lanes, four bytes each, they are four requests in eight, and a fifth of the bytes
// took a third of the time: a batch of 32 sequences of up to 8000 positions, heads of 128, 69 us for reading alone, 47 so.)
template <int kHs>
struct ScaleRows {
    static constexpr int kWords = kHs / kKv4Group, kRowBytes = 4 * kWords, kLdsBytes = 64 * kRowBytes;
    typedef uint32_t Row __attribute__((ext_vector_type(kWords)));
    Row row;
    __device__ __forceinline__ void load(const uint32_t* scales_of_head, int pos) {
        row = __builtin_nontemporal_load(reinterpret_cast<const Row*>(reinterpret_cast<const char*>(scales_of_head) + static_cast<uint32_t>(pos) * kRowBytes));
    }
    __device__ __forceinline__ void put(char* lds) const { *reinterpret_cast<Row*>(lds + lane_id() * kRowBytes) = row; }
    // scale and lowest value of row `row` for the values of a Piece
    static __device__ __forceinline__ uint32_t get(const char* lds, int row, int part) {
        return *reinterpret_cast<const uint32_t*>(lds + row * kRowBytes + part * kWords / 4 * 4);
    }
};

// Q of a tile as B operands: column lane % 16, the values that a K piece's words have; heads and remainders.  Heads of 128 have them in LDS, the
// same for all wavefronts of a workgroup: in registers they are 32 of them, and with 168 for three wavefronts to a SIMD the loop spills, whose
// reloads wait for the K and V rows that are on their way.
template <int kHs>
struct Queries {
    static constexpr int kWords = kHs / 32;
    static constexpr bool kInLds = kHs == 128;
    static constexpr int kLdsBytes = kInLds ? 2 * kWords * 16 * kWave : 0;
    half8_t held[kInLds ? 1 : 2 * kWords];  // [word][head, remainder]
    const half8_t* shared;
    // wave, waves: this wavefront's share of the work (a barrier has to follow)
    __device__ __forceinline__ void load(const float* row, int part, char* lds, int wave, int waves) {
        half8_t* to = reinterpret_cast<half8_t*>(lds) + lane_id();
        shared = to;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if (kInLds && i % waves != wave) continue;
            const float* from = row + part * kWords * 8 + 8 * i;
            const floatx4 a = as_float4(load16(from)), b = as_float4(load16(from + 4));
            half8_t high, low;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = e < 4 ? a[e & 3] : b[e & 3];
                high[e] = static_cast<half_t>(v);
                low[e] = static_cast<half_t>(v - static_cast<float>(high[e]));
            }
            if constexpr (kInLds) {
                to[2 * i * kWave] = high;
                to[(2 * i + 1) * kWave] = low;
            } else {
                held[2 * i] = high;
                held[2 * i + 1] = low;
            }
        }
    }
    // scores of n x 16 positions: lane: column lane % 16, positions 4 (lane / 16) ..
    template <int n>
    __device__ __forceinline__ void scores(const Kv4Reader& read, const Piece<kHs>* k, floatx4* st) const {
#pragma unroll
        for (int t = 0; t < n; ++t) st[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            half8_t high, low;
            if constexpr (kInLds) {
                high = shared[2 * i * kWave];
                low = shared[(2 * i + 1) * kWave];
            } else {
                high = held[2 * i];
                low = held[2 * i + 1];
            }
#pragma unroll
            for (int t = 0; t < n; ++t) {
                const half8_t kv = k[t].values(read, i);
                st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, high, st[t], 0, 0, 0);
                st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, low, st[t], 0, 0, 0);
            }
        }
    }
};

// Which row a column of a tile is.
struct Column {
    int in_tile, token, head;
    bool valid;
    __device__ __forceinline__ Column(const AttendJob& job, int tile, int column) {
        const int tokens = job.tokens();
        in_tile = static_cast<int>(column * job.per_shared >> 16);
        head = column - in_tile * job.shared;
        token = tile * tokens + in_tile;
        valid = in_tile < tokens && token < job.n_q;
        token = min(token, min(tile * tokens + tokens, job.n_q) - 1);
    }
    __device__ __forceinline__ size_t at(const AttendJob& job, int s, int kvh) const {
        return (static_cast<size_t>(s) * job.n_q + token) * job.n_kv_heads * job.shared + kvh * job.shared + head;
    }
};

// A share of a sequence's positions for a tile of rows and a KV head; its wavefronts take steps of kStep positions in turn and merge at
// the end.  Registers: four wavefronts to a SIMD for heads of 64, three for 128, without spills.
template <int kHs, int kWaves>
__global__ __launch_bounds__(kWave * kWaves, kHs == 64 ? 4 : 3) void attend_kernel(AttendJob job) {
    constexpr int kDTiles = kHs / 16, kWords = kHs / 32, kRowBytes = 2 * kHs, kThreads = kWave * kWaves;
    constexpr int kPad = kHs + 4, kPart = kRows * kPad + 2 * kRows;  // floats a wavefront leaves for the merge
    constexpr int kWaveBytes = kPart * 4 + ScaleRows<kHs>::kLdsBytes;
    static_assert(kPart * 4 >= kStep * kRowBytes && kWaveBytes % 16 == 0, "V rows of a step");
    extern __shared__ __align__(16) char lds[];
    const int lane = lane_id(), wave = wave_index(), column = lane & 15, part = lane >> 4;
    // (Heads of sequences first, then a head's tiles, then the shares: whatever number of the shares there are, the workgroups that have one are
    // dealt out evenly over the dies, and the tiles of a head, which read the same rows, go to the same die where the heads
    // are a multiple of its number.)
    const int head = static_cast<int>(blockIdx.x % job.heads), rest = static_cast<int>(blockIdx.x / job.heads);
    const int kvh = head % job.n_kv_heads, s = head / job.n_kv_heads, tile = rest % job.tiles, split = rest / job.tiles;
    const int tokens = job.tokens(), start = job.start_of(s);
    const int all_end = job.end_of(start, job.n_q - 1);
    const int shares = job.shares_of(all_end);
    if (split >= shares) return;
    const int end = job.end_of(start, min(tile * tokens + tokens, job.n_q) - 1);  // the tile's last row attends to [0, end)
    const bool only = shares == 1;                                               // (uniform over the sequence: no merge)
    // A workgroup's steps are one for each of its wavefronts in every round of all shares' workgroups: what they read at a time is one
    // stretch of the head's rows.
    const int first = (split * kWaves + wave) * kStep, stride = shares * kWaves * kStep;
    const Column mine(job, tile, column);
    const int my_end = job.end_of(start, mine.token), first_end = job.end_of(start, tile * tokens);
    const size_t head_rows = (static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.seq_len;
    const uint32_t* codes[2];
    const uint32_t* scales[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        codes[w] = job.cache.codes[w] + head_rows * (kHs / 8);
        scales[w] = job.cache.scales[w] + head_rows * (kHs / kKv4Group);
    }
    // K and V of a step travel while the step before is worked on, each requested as soon as its registers are free.  (Also behind the last
    // step, whose requests are the last row's again: were they conditional, a wait for one would have to be a wait for all.)
    Piece<kHs> k[2], v[2];
    auto request = [&](Piece<kHs>(&to)[2], int which, int p0) {
#pragma unroll
        for (int t = 0; t < 2; ++t) to[t].load(codes[which], min(p0 + 16 * t + column, end - 1), part);
    };
    ScaleRows<kHs> pairs;
    char* pairs_lds = lds + wave * kWaveBytes + kPart * 4;
    const uint32_t* my_scales = lane < 32 ? scales[0] : scales[1];
    auto request_pairs = [&](int p0) { pairs.load(my_scales, min(p0 + (lane & 31), end - 1)); };
    if (first < end) {
        request_pairs(first);
        request(k, 0, first);
        request(v, 1, first);
    }
    Queries<kHs> q;
    q.load(job.q + mine.at(job, s, kvh) * kHs, part, lds + kWaves * kWaveBytes, wave, kWaves);
    if constexpr (Queries<kHs>::kInLds) __syncthreads();
    const Kv4Reader read;

    floatx4 o[kDTiles];
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) o[dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const float scale = 1.44269504088896341f / sqrtf(static_cast<float>(kHs));
    float top = 0.0f, lsum = 0.0f;  // (the sum over this lane's own positions)
    bool seen = false;              // the row has attended to something: top is a score less kLift
    float minus_one = -1.0f;
    asm("" : "+v"(minus_one));

    // V rows of a step, in this wavefront's own LDS: 16-byte pieces in an order that keeps writes free of bank conflicts, and transposing reads of
    // heads of 64.  (Of heads of 128 half a wavefront reads a pair of pieces of eight rows, and rows four apart have theirs in the same banks: two cycles
    // for one, 41 % of the LDS's in a batch of 32 sequences.)
    char* values = lds + wave * kWaveBytes;
    auto swizzle = [](int row) { return kHs == 64 ? 2 * ((row >> 1) & 3) : 4 * (row & 3) + ((row >> 2) & 3); };
    int v_at[kDTiles], v_to[kWords];  // (of the first sixteen positions; the others are 16 rows further, in the same order)
    {
        const int row = 4 * part + ((lane & 15) >> 2);
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt) v_at[dt] = row * kRowBytes + 16 * ((2 * dt + ((lane & 3) >> 1)) ^ swizzle(row)) + 8 * (lane & 1);
#pragma unroll
        for (int i = 0; i < kWords; ++i) v_to[i] = column * kRowBytes + 16 * ((kWords * part + i) ^ swizzle(column));
    }

    // (stored behind the step's requests of K and V, so that those do not wait for the stores)
    const bool keeps = job.scores != nullptr && mine.valid;
    float* my_scores = job.scores + (static_cast<size_t>(head) * job.steps * job.rows + min(column, job.rows - 1)) * kStep + 4 * part;
    for (int p0 = first; p0 < end; p0 += stride) {
        const bool partly = p0 + kStep > first_end;   // (uniform) some row does not attend to the whole step
        pairs.put(pairs_lds);
        request_pairs(p0 + stride);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            k[t].pair = ScaleRows<kHs>::get(pairs_lds, 16 * t + column, part);
            v[t].pair = ScaleRows<kHs>::get(pairs_lds, 32 + 16 * t + column, part);
        }
        floatx4 st[2];
        q.template scores<2>(read, k, st);
        request(k, 0, p0 + stride);
        // V rows behind the tile's last position are zero: a weight of zero does not keep an infinity or NaN out.
        if (partly) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (p0 + 16 * t + column >= end) v[t].pair = 0u;
        }
        const bool odd = __builtin_amdgcn_ballot_w64(v[0].may_be_nonfinite() || v[1].may_be_nonfinite()) != 0ull;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < kWords; ++i) *reinterpret_cast<half8_t*>(values + v_to[i] + 16 * t * kRowBytes) = v[t].values(read, i);
        request(v, 1, p0 + stride);
        if (keeps) {
#pragma unroll
            for (int t = 0; t < 2; ++t) *reinterpret_cast<floatx4*>(my_scores + p0 * job.rows + 16 * t) = st[t];
        }
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
        const bool moves = step_top > (seen ? top + (kLift + kSlack) : -INFINITY);
        if (__builtin_amdgcn_ballot_w64(moves) != 0ull) {  // (uniform)
            const float to = moves ? step_top - kLift : top;
            const float corr = __builtin_amdgcn_exp2f(seen ? top - to : 0.0f);  // (nothing to rescale before a row's first step)
            top = to;
            lsum *= corr;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) o[dt] *= corr;
            seen = seen || moves;
        }
        half8_t ph, pl;
        float step_sum = 0.0f;  // (of its own, so that the running sum is rounded once a step)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float p_0 = __builtin_amdgcn_exp2f(fmaf(st[e >> 2][e & 3], scale, -top));
            const float p_1 = __builtin_amdgcn_exp2f(fmaf(st[e >> 2][(e & 3) + 1], scale, -top));
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
        auto values_of = [&](int dt) {
            union {
                short4_t half[2];
                half8_t whole;
            } vf;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                vf.half[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(values + v_at[dt] + 16 * t * kRowBytes));
            return vf.whole;
        };
        if (odd) {
            // (uniform) An infinity or NaN, perhaps, among the step's V rows: one token after the other, with the rows behind it cleared; a
            // lane's output is its own token's.  The weights' remainders, of either sign, meet the finite values only.
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) {
                const half8_t all = values_of(dt);
                for (int token = 0; token < tokens; ++token) {
                    const int token_end = job.end_of(start, tile * tokens + token) - p0 - 4 * part;
                    half8_t x = all;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((e & 3) + 16 * (e >> 2) >= token_end) x[e] = static_cast<half_t>(0.0f);
                    floatx4 with = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph, o[dt], 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (!(fabsf(static_cast<float>(x[e])) < INFINITY)) x[e] = static_cast<half_t>(0.0f);
                    with = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl, with, 0, 0, 0);
                    if (mine.in_tile == token) o[dt] = with;
                }
            }
        } else {
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) {
                const half8_t x = values_of(dt);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph, o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl, o[dt], 0, 0, 0);
            }
        }
    }
    lsum = rows_sum(lsum);
    if (!seen) top = -INFINITY;

    // The wavefronts meet in LDS: four neighbouring lanes add four values of a row, each a quarter of the wavefronts in their order.  Those that
    // had no step have left nothing and are not read.
    const int parts = min(max((end - split * kWaves * kStep + kStep - 1) / kStep, 1), kWaves);
    constexpr int kPartStep = kWaveBytes / 4;
    float* all = reinterpret_cast<float*>(lds);
    if (wave < parts) {
        float* my_part = all + wave * kPartStep;
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt) *reinterpret_cast<floatx4*>(my_part + column * kPad + 16 * dt + 4 * part) = o[dt];
        if (part == 0) {
            my_part[kRows * kPad + column] = top;
            my_part[kRows * kPad + kRows + column] = lsum;
        }
    }
    __syncthreads();
    const size_t slot = ((static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.tiles + tile) * job.splits + split;
    constexpr int kFours = kHs / 4;
    const int used = min(tokens, job.n_q - tile * tokens) * job.shared;  // rows there are
    const int quarter = lane & 3;
    // (whole wavefronts go round: the lanes of a quarter are all here)
    for (int i = static_cast<int>(threadIdx.x) / 4; i < (used * kFours + 15) / 16 * 16; i += kThreads / 4) {
        const bool there = i < used * kFours;
        const int row = there ? i / kFours : 0, four = i % kFours;
        constexpr int kMine = kWaves / 4;
        float weight[kMine], all_top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int w = quarter * kMine + j;
            weight[j] = w < parts ? all[w * kPartStep + kRows * kPad + row] : -INFINITY;
            all_top = fmaxf(all_top, weight[j]);
        }
        all_top = fmaxf(all_top, dpp_move<kDppXor1>(all_top));
        all_top = fmaxf(all_top, dpp_move<kDppXor2>(all_top));
        const float reference = all_top == -INFINITY ? 0.0f : all_top;  // (nothing seen, or no score was a number)
        floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int w = quarter * kMine + j;
            if (w >= parts) break;
            weight[j] = __builtin_amdgcn_exp2f(weight[j] - reference);
            total = fmaf(all[w * kPartStep + kRows * kPad + kRows + row], weight[j], total);
            const floatx4 a = *reinterpret_cast<const floatx4*>(all + w * kPartStep + row * kPad + 4 * four);
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[u] = fmaf(a[u], weight[j], sum[u]);
        }
        total += dpp_move<kDppXor1>(total);
        total += dpp_move<kDppXor2>(total);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            sum[u] += dpp_move<kDppXor1>(sum[u]);
            sum[u] += dpp_move<kDppXor2>(sum[u]);
        }
        if (!there || quarter != 0) continue;
        if (only) {
            const Column its(job, tile, row);
            const bool any = job.end_of(start, its.token) > 0;
            const float inverse = 1.0f / total;
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[u] = any ? sum[u] * inverse : 0.0f;
            *reinterpret_cast<floatx4*>(job.out + its.at(job, s, kvh) * kHs + 4 * four) = sum;
        } else {
            *reinterpret_cast<floatx4*>(job.partials + (slot * job.rows + row) * kHs + 4 * four) = sum;
        }
        if (four == 0) job.stats[slot * job.rows + row] = make_float2(all_top, total);
    }
}

// What is left once every share has been walked: the first blocks, `accounts` of them, add up the weights of the positions, the others (where there
// are shares to merge) merge a row with each wavefront.
constexpr int kFinishWaves = 4, kFinishThreads = kWave * kFinishWaves;

// Maximum and 1 / sum of a tile's rows, each in the lanes that have its column: the shares' in four parts, which meet across those lanes.
struct Sums {
    float top, inverse;
    __device__ __forceinline__ void load(const AttendJob& job, int head, int tile, bool valid, int active) {
        const int column = lane_id() & 15, part = lane_id() >> 4;
        const float2* stats = job.stats + (static_cast<size_t>(head) * job.tiles + tile) * job.splits * job.rows + column;
        float all = -INFINITY, total = 0.0f;
        for (int i0 = 0; i0 < active; i0 += 16) {
            float2 st[4];
            float highest = all;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = i0 + 4 * j + part;
                st[j] = valid && at < active ? stats[at * job.rows] : make_float2(-INFINITY, 0.0f);
                highest = fmaxf(highest, st[j].x);
            }
            const float reference = highest == -INFINITY ? 0.0f : highest;
            total *= __builtin_amdgcn_exp2f(all - reference);
#pragma unroll
            for (int j = 0; j < 4; ++j) total = fmaf(st[j].y, __builtin_amdgcn_exp2f(st[j].x - reference), total);
            all = highest;
        }
        const float highest = rows_max(all);
        top = highest == -INFINITY ? 0.0f : highest;
        inverse = 1.0f / rows_sum(total * __builtin_amdgcn_exp2f(all - top));
    }
};

// kKept: the account is made from the scores that the shares have kept; else from K again.
template <int kHs, bool kKept>
__global__ __launch_bounds__(kFinishThreads) void finish_kernel(AttendJob job, int accounts, int span) {
    constexpr int kFours = kHs / 4, kSlices = kWave / kFours, kPieces = 4, kOfWave = 16 * kPieces;
    constexpr int kQueryBytes = Queries<kHs>::kLdsBytes > 0 ? Queries<kHs>::kLdsBytes : 16;
    __shared__ __align__(16) char scale_lds[kFinishWaves][ScaleRows<kHs>::kLdsBytes];
    __shared__ __align__(16) char q_lds[kFinishWaves][kQueryBytes];
    __shared__ float of_waves[kFinishWaves][kOfWave];
    const int lane = lane_id(), wave = wave_index(), column = lane & 15, part = lane >> 4;
    const int head = static_cast<int>(blockIdx.x % job.heads), block = static_cast<int>(blockIdx.x / job.heads);
    const int kvh = head % job.n_kv_heads, s = head / job.n_kv_heads, start = job.start_of(s), tokens = job.tokens();
    const int all_end = job.end_of(start, job.n_q - 1);
    const int active = job.shares_of(all_end);
    if (block >= accounts) {
        // A wavefront to a row: its lanes have four values each of every kSlices-th share.
        if (active == 1) return;
        const int index = (block - accounts) * kFinishWaves + wave;
        if (index >= job.tiles * job.rows) return;
        const int tile = index / job.rows, row = index % job.rows;
        const Column its(job, tile, row);
        if (!its.valid) return;
        const size_t slot = (static_cast<size_t>(head) * job.tiles + tile) * job.splits;
        const int slice = lane / kFours, four = lane % kFours;
        const float2 st = lane < active ? job.stats[(slot + lane) * job.rows + row] : make_float2(-INFINITY, 0.0f);
        const float* from = job.partials + (slot * job.rows + row) * kHs + 4 * four;
        floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        float weight = 0.0f, total = 0.0f;
        // (the shares' outputs are requested along with their sums, kAtOnce rounds of them; a share that the row does not attend to has left none)
        constexpr int kAtOnce = 8;
        for (int i0 = 0; i0 < active; i0 += kAtOnce * kSlices) {
            floatx4 a[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (i0 + i * kSlices >= active) break;  // (uniform)
                a[i] = *reinterpret_cast<const floatx4*>(from + static_cast<size_t>(min(i0 + i * kSlices + slice, active - 1)) * job.rows * kHs);
            }
            if (i0 == 0) {
                float top = wave_max(st.x);
                if (top == -INFINITY) top = 0.0f;
                weight = __builtin_amdgcn_exp2f(st.x - top);
                total = wave_sum(st.y * weight);
                if (st.x == -INFINITY && st.y == 0.0f) weight = -1.0f;  // (lanes without a share too)
            }
            float w[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) w[i] = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (i0 + i * kSlices + slice), __float_as_int(weight)));
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (i0 + i * kSlices >= active) break;
                if (w[i] >= 0.0f)
#pragma unroll
                    for (int u = 0; u < 4; ++u) sum[u] = fmaf(a[i][u], w[i], sum[u]);
            }
        }
        const bool any = job.end_of(start, its.token) > 0;
        const float inverse = 1.0f / total;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            sum[u] = kSlices == 4 ? rows_sum(sum[u]) : halves_sum(sum[u]);
            sum[u] = any ? sum[u] * inverse : 0.0f;
        }
        if (slice == 0) *reinterpret_cast<floatx4*>(job.out + its.at(job, s, kvh) * kHs + 4 * four) = sum;
        return;
    }
    const int p_first = block * span;
    if (p_first >= all_end) return;
    float* mass = job.mass + (static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.seq_len;
    const float scale = 1.44269504088896341f / sqrtf(static_cast<float>(kHs));
    Sums sums;
    if constexpr (kKept) {
        const float* scores = job.scores + static_cast<size_t>(head) * job.steps * job.rows * kStep;
        // of a row whose lane has its sums: what a score adds to position p
        auto weight = [&](float score, int row, int p, int row_end) {
            const float top = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sums.top), row));
            const float inverse = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sums.inverse), row));
            return p < row_end ? __builtin_amdgcn_exp2f(fmaf(score, scale, -top)) * inverse : 0.0f;
        };
        // Four positions to a lane, four rows at a time, the next of them on their way.
        typedef float Unaligned4 __attribute__((ext_vector_type(4), aligned(4)));
        constexpr int kAt = 4, kOnce = 4 * kWave;
        const int p_end = min(p_first + span, all_end);
        floatx4 sc[kAt], now[kAt];
        auto request = [&](int p0, int c0) {
            const int at = min(p0 + 4 * lane, job.steps * kStep - 4);
            const float* from = scores + static_cast<size_t>(at / kStep) * job.rows * kStep + at % kStep;
#pragma unroll
            for (int c = 0; c < kAt; ++c) sc[c] = *reinterpret_cast<const floatx4*>(from + min(c0 + c, job.rows - 1) * kStep);
        };
        int p0 = p_first + kOnce * wave;
        if (p0 >= p_end) return;  // (no barrier ahead)
        request(p0, 0);
        sums.load(job, head, 0, Column(job, 0, column).valid, active);
        while (p0 < p_end) {  // (uniform in the wavefront)
            const int p = p0 + 4 * lane;
            const bool whole = p + 4 <= all_end;
            floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f}, before = sum;
            if (whole) before = *reinterpret_cast<const Unaligned4*>(mass + p);
            p0 += kOnce * kFinishWaves;
            for (int c0 = 0; c0 < job.rows; c0 += kAt) {
#pragma unroll
                for (int c = 0; c < kAt; ++c) now[c] = sc[c];
                if (c0 + kAt < job.rows) request(p - 4 * lane, c0 + kAt);
                else if (p0 < p_end) request(p0, 0);
#pragma unroll
                for (int c = 0; c < kAt; ++c) {
                    if (c0 + c >= job.rows) break;
                    const int row_end = job.end_of(start, static_cast<int>((c0 + c) * job.per_shared >> 16));
#pragma unroll
                    for (int u = 0; u < 4; ++u) sum[u] += weight(now[c][u], c0 + c, p + u, row_end);
                }
            }
            if (whole) *reinterpret_cast<Unaligned4*>(mass + p) = before + sum;
            else
                for (int u = 0; u < 4; ++u)
                    if (p + u < all_end) mass[p + u] += sum[u];
        }
    } else {
        const size_t head_rows = (static_cast<size_t>(s) * job.n_kv_heads + kvh) * job.seq_len;
        // One tile: the wavefronts take the positions in turn.  Several: each position's tiles (one after the other in every wavefront, what counts
        // is the time of a tile's requests: 16 rows of 4 sequences of up to 3000 positions, heads of 64, 18 us and 14).
        const bool by_tiles = job.tiles > 1;
        const int p0 = p_first + (by_tiles ? 0 : kOfWave * wave);
        const Kv4Reader read;
        Piece<kHs> k[kPieces];
        ScaleRows<kHs> pairs;
        char* pairs_lds = scale_lds[wave];
        pairs.load(job.cache.scales[0] + head_rows * (kHs / kKv4Group), min(p0 + lane, all_end - 1));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) k[i].load(job.cache.codes[0] + head_rows * (kHs / 8), min(p0 + 16 * i + column, all_end - 1), part);
        pairs.put(pairs_lds);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) k[i].pair = ScaleRows<kHs>::get(pairs_lds, 16 * i + column, part);
        floatx4 sum[kPieces];  // of this lane's column, over the tiles
#pragma unroll
        for (int i = 0; i < kPieces; ++i) sum[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int tile = by_tiles ? wave : 0; tile < job.tiles; tile += by_tiles ? kFinishWaves : 1) {
            if (job.end_of(start, min(tile * tokens + tokens, job.n_q) - 1) <= p0) continue;  // (uniform in the wavefront)
            const Column mine(job, tile, column);
            const int my_end = mine.valid ? job.end_of(start, mine.token) : 0;
            Queries<kHs> q;
            q.load(job.q + mine.at(job, s, kvh) * kHs, part, q_lds[wave], 0, 1);
            sums.load(job, head, tile, mine.valid, active);
            // (uniform) a row does not attend to all of the positions, or there is no row
            const bool partly = p0 + kOfWave > job.end_of(start, tile * tokens) || job.rows < kRows || (tile + 1) * tokens > job.n_q;
#pragma unroll
            for (int i = 0; i < kPieces; i += 2) {
                floatx4 st[2];
                q.template scores<2>(read, k + i, st);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float w = __builtin_amdgcn_exp2f(fmaf(st[t][e], scale, -sums.top)) * sums.inverse;
                        if (partly) w = p0 + 16 * (i + t) + 4 * part + e < my_end ? w : 0.0f;
                        sum[i + t][e] += w;
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[i][e] = row16_sum(sum[i][e]);
            const float mine = column == 0 ? sum[i][0] : column == 1 ? sum[i][1] : column == 2 ? sum[i][2] : sum[i][3];
            if (column < 4) of_waves[wave][16 * i + 4 * part + column] = mine;
        }
        __syncthreads();
        const int p = p_first + static_cast<int>(threadIdx.x);
        if (static_cast<int>(threadIdx.x) >= span || p >= all_end) return;
        float total = 0.0f;
        if (by_tiles) {
#pragma unroll
            for (int w = 0; w < kFinishWaves; ++w) total += of_waves[w][threadIdx.x];
        } else {
            total = of_waves[wave][lane];
        }
        mass[p] += total;
    }
}

int tiles_of(int n_q, int shared) { return (n_q + kRows / shared - 1) / (kRows / shared); }

// Shares a sequence's positions are cut into at most, the least positions of one, the wavefronts to one, and how many of them run at once. Few heads:
// 8 wavefronts to a share, for half the steps of each (one sequence of 8 KV heads of 64, us at 500 / 1000 / 8000 positions: 6.4 / 9.3 / 9.4, 6.8 /
// 9.7 / 9.8 with 4 and 6.7 / 9.6 / 9.8 with 16; of 128: 8.2 / 10.9 / 11.4, 9.4 / 12.2 / 12.6 with 4).  512 positions at least: 256 or 1024 give one
// sequence of 16001 10.1 or 9.7 us for 8.0, and more or fewer shares to merge.
struct Split {
    int splits, least, waves, workgroups;
    size_t most, rounds;  // shares of a sequence by its positions; of all tiles
};
Split split_of(const lpp_kv4_shape& shape, int tiles) {
    const long long heads = static_cast<long long>(shape.n_seqs) * shape.n_kv_heads * tiles;
    Split s;
    s.waves = heads * 4 > compute_units() ? 4 : 8;
    s.least = 512;
    s.workgroups = compute_units() * (shape.head_size == 64 ? 16 / s.waves : s.waves == 8 ? 1 : 3);  // (by registers, and LDS for the heads of 128)
    const int most = (shape.seq_len + s.least - 1) / s.least;
    s.splits = most < kMaxSplits ? most : kMaxSplits;
    s.most = s.splits;
    // (no more workgroups than 16 rounds of them, most of which would find no share)
    s.rounds = 16ull * s.workgroups;
    const long long rounds = 16ll * s.workgroups / heads;
    if (s.splits > rounds) s.splits = static_cast<int>(rounds > 1 ? rounds : 1);
    return s;
}

// What the workspace holds.  Scores kept for the account are 4 bytes for every position and row; made from K again they cost its bytes and the
// products (32 sequences of up to 8000 positions, 4 rows to a KV head of 128: 49 us more than without an account, and 10 so).  Not of several tiles,
// whose scores are many times a layer (16 rows of 32 heads, 4 sequences of up to 3000 positions, heads of 64: 27.5 us for 25.5), and only where the
// workspace gets no larger than partial results of kMaxSplits shares would make it: up to about 14900 positions with four rows to a KV head of 64,
// 3680 with sixteen.
// `bytes` is no less than that of any call of fewer sequences, positions, heads or rows, whose layout may take more than this one's (scores that this one
// does not keep; shares, whose number is rounded down to what runs at once): one workspace serves them all.
struct Workspace {
    size_t stats, partials, scores;  // floats
    int rows, steps;
    size_t bytes;
    Workspace(const lpp_kv4_shape& shape, int n_q, int shared, int tiles, const Split& split) {
        const size_t heads = static_cast<size_t>(shape.n_seqs) * shape.n_kv_heads, all_tiles = heads * tiles;
        rows = (n_q < kRows / shared ? n_q : kRows / shared) * shared;
        steps = (shape.seq_len + kStep - 1) / kStep;
        const size_t limit = heads * kMaxSplits * kRows * (shape.head_size + 2), of_scores = heads * steps * kStep;
        const auto sums = [](size_t slots) { return (slots * 2 + 3) / 4 * 4; };
        const size_t slots = all_tiles * split.splits * rows;
        stats = sums(slots);
        partials = slots * shape.head_size;
        scores = tiles == 1 && stats + partials + of_scores * rows <= limit ? of_scores * rows : 0;
        // (split_of's numbers before they are rounded: as many shares as positions make, within `rounds`, and all rows that a tile has room for)
        const size_t most_rows = static_cast<long long>(n_q) * shared < kRows ? static_cast<size_t>(n_q) * shared : kRows;
        size_t most = all_tiles * split.most < split.rounds ? all_tiles * split.most : split.rounds;
        if (most < all_tiles) most = all_tiles;
        const size_t shares = sums(most * most_rows) + most * most_rows * shape.head_size, kept = shares + of_scores * most_rows;
        const size_t with_scores = kept < limit ? kept : limit;
        bytes = (shares > with_scores ? shares : with_scores) * sizeof(float);
    }
};

template <int kHs, int kWaves>
lpp_status launch_attend(const AttendJob& job, dim3 grid) {
    constexpr int kLds = kWaves * ((kRows * (kHs + 4) + 2 * kRows) * 4 + ScaleRows<kHs>::kLdsBytes) + Queries<kHs>::kLdsBytes;
    const auto kernel = &attend_kernel<kHs, kWaves>;
    if constexpr (kLds > 64 * 1024) {
        static bool sized[64] = {};
        LPP_TRY(tell_lds(reinterpret_cast<const void*>(kernel), kLds, sized));
    }
    hipLaunchKernelGGL(kernel, grid, dim3(kWave * kWaves), kLds, stream(), job);
    LPP_CHECK_LAUNCH("attend_kernel");
    return LPP_OK;
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
    *bytes = Workspace(*shape, n_q, n_heads / shape->n_kv_heads, tiles, split_of(*shape, tiles)).bytes;
    return LPP_OK;
}

lpp_status lpp_kv4_attention(float* d_out, const float* d_q, const void* d_cache, const lpp_kv4_shape* shape, int layer, int n_heads, int n_q,
                             const int* d_starts, float* d_mass, void* d_workspace, size_t workspace_bytes) {
    using namespace lpp;
    LPP_TRY(kv4_check_cache("lpp_kv4_attention", d_cache, shape, layer));
    LPP_TRY(check("lpp_kv4_attention", shape, n_heads, n_q));
    LPP_REQUIRE(d_out && d_q && d_starts && d_workspace, "lpp_kv4_attention: null pointer");
    const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    LPP_REQUIRE(aligned(d_out) && aligned(d_q) && aligned(d_workspace),
                "lpp_kv4_attention: d_out, d_q and d_workspace must start at multiples of 16 bytes");
    size_t need = 0;
    LPP_TRY(lpp_kv4_attention_workspace(shape, n_heads, n_q, &need));
    LPP_REQUIRE(workspace_bytes >= need, "lpp_kv4_attention: a workspace of %zu bytes, %zu are needed", workspace_bytes, need);
    const size_t rows_bytes = static_cast<size_t>(shape->n_seqs) * n_q * n_heads * shape->head_size * 4;
    LPP_REQUIRE(!ranges_overlap(d_out, rows_bytes, d_q, rows_bytes), "lpp_kv4_attention: d_out overlaps d_q");
    LPP_REQUIRE(!ranges_overlap(d_workspace, need, d_q, rows_bytes) && !ranges_overlap(d_workspace, need, d_out, rows_bytes) &&
                    !ranges_overlap(d_workspace, need, d_cache, kv4_bytes(*shape)),
                "lpp_kv4_attention: the workspace overlaps q, out or the cache");
    const size_t mass_bytes = d_mass != nullptr ? kv4_layer_rows(*shape) * shape->n_layers * 4 : 0;
    LPP_REQUIRE(mass_bytes == 0 || (!ranges_overlap(d_mass, mass_bytes, d_workspace, need) && !ranges_overlap(d_mass, mass_bytes, d_q, rows_bytes) &&
                                    !ranges_overlap(d_mass, mass_bytes, d_out, rows_bytes) && !ranges_overlap(d_mass, mass_bytes, d_cache, kv4_bytes(*shape))),
                "lpp_kv4_attention: d_mass overlaps the workspace, q, out or the cache");
    LPP_REQUIRE(!ranges_overlap(d_out, rows_bytes, d_cache, kv4_bytes(*shape)), "lpp_kv4_attention: d_out overlaps the cache");
    const size_t starts_bytes = static_cast<size_t>(shape->n_seqs) * 4;
    LPP_REQUIRE(!ranges_overlap(d_starts, starts_bytes, d_out, rows_bytes) && !ranges_overlap(d_starts, starts_bytes, d_workspace, need) &&
                    (mass_bytes == 0 || !ranges_overlap(d_starts, starts_bytes, d_mass, mass_bytes)),
                "lpp_kv4_attention: d_starts overlaps out, the workspace or d_mass");
    AttendJob job;
    job.out = d_out;
    job.q = d_q;
    job.cache = kv4_layer(d_cache, *shape, layer);
    job.starts = d_starts;
    job.mass = d_mass != nullptr ? d_mass + kv4_layer_rows(*shape) * layer : nullptr;
    job.heads = static_cast<unsigned>(shape->n_seqs) * shape->n_kv_heads;
    job.n_seqs = shape->n_seqs;
    job.n_q = n_q;
    job.n_kv_heads = shape->n_kv_heads;
    job.shared = n_heads / shape->n_kv_heads;
    job.seq_len = shape->seq_len;
    job.tiles = tiles_of(n_q, job.shared);
    const Split split = split_of(*shape, job.tiles);
    job.splits = split.splits;
    job.least = split.least;
    // Of many heads a quarter more shares than run at once: they are of unequal length, and the last to begin are not the last to end.  us for 1 /
    // 1.25 / 1.5 / 2 times as many, heads of 128, ragged: 32 sequences of up to 8000 positions 62 / 59 / 56 / 58, 64 of 4000 60 / 58 / 58 / 59; 32 of
    // 4000 alike 43 / 41.  Of few heads no more than run at once: 4 sequences of 8000 alike 17 / 23.
    job.per_workgroup = static_cast<float>(shape->n_kv_heads) * job.tiles / (split.waves == 4 ? 1.25f * split.workgroups : split.workgroups);
    job.per_shared = (65536u + job.shared - 1) / job.shared;
    const Workspace parts(*shape, n_q, job.shared, job.tiles, split);
    job.rows = parts.rows;
    job.steps = parts.steps;
    job.stats = static_cast<float2*>(d_workspace);
    job.partials = static_cast<float*>(d_workspace) + parts.stats;
    job.scores = d_mass != nullptr && parts.scores > 0 ? job.partials + parts.partials : nullptr;
    const long long groups = static_cast<long long>(job.heads) * job.tiles * job.splits;
    LPP_REQUIRE(groups * dev::kWave * split.waves < (1ll << 32),
                "lpp_kv4_attention: %u sequences times KV heads and %d rows are too many for a launch", job.heads, n_q);
    const int merges = job.splits > 1 ? (job.tiles * job.rows + kFinishWaves - 1) / kFinishWaves : 0;
    // The positions of one of the account's blocks.  From kept scores of one tile: as many rounds of 1024, up to 8, as leave four blocks to a compute
    // unit.
    const bool kept = job.scores != nullptr;
    int span = job.tiles > 1 ? kWave : (kept ? 4 : 1) * kFinishThreads;
    if (kept) {
        const long long each = (static_cast<long long>(shape->seq_len) + span - 1) / span * job.heads / (4 * compute_units());
        span *= each < 1 ? 1 : each < 8 ? static_cast<int>(each) : 8;
    }
    const int accounts = d_mass != nullptr ? (shape->seq_len + span - 1) / span : 0, blocks = merges + accounts;
    LPP_REQUIRE(static_cast<long long>(blocks) * job.heads * kFinishThreads < (1ll << 32),
                "lpp_kv4_attention: %u sequences times KV heads of %d positions are too many for a launch", job.heads, shape->seq_len);
    // (nothing is refused from here on)
    const dim3 grid(static_cast<unsigned>(groups));
    if (shape->head_size == 64)
        LPP_TRY(split.waves == 8 ? (launch_attend<64, 8>(job, grid)) : (launch_attend<64, 4>(job, grid)));
    else
        LPP_TRY(split.waves == 8 ? (launch_attend<128, 8>(job, grid)) : (launch_attend<128, 4>(job, grid)));
    if (blocks > 0) {
        const auto kernel = shape->head_size == 64 ? (kept ? &finish_kernel<64, true> : &finish_kernel<64, false>)
                                                   : (kept ? &finish_kernel<128, true> : &finish_kernel<128, false>);
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks) * job.heads), dim3(kFinishThreads), 0, stream(), job, accounts, span);
        LPP_CHECK_LAUNCH("finish_kernel");
    }
    return LPP_OK;
}

}  // extern "C"
