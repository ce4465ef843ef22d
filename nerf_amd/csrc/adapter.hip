// adapter.hip — linear layers with weights shared by all rows and a low-rank
// adapter of every group of rows beside them (include/nerf_ext.h,
// nerf_ext_adapter_linear_*).
//
//   forward:   m_i = A_g x_i,  z_i = W x_i + b + s_g B_g m_i,  y_i = act(z_i) + r_i
//   backward:  n_i = s_g B_g^T d_i,  g_i = d_i W + n_i A_g + a_i,  dx = g,  dpre = g act'(pre),
//              dA_g = sum_i n_i x_i^T,  dB_g = s_g sum_i d_i m_i^T
//
// m and n (rank values a row, 32 bits) are a grouped product of their own; the
// shared product then goes over all rows in tiles of any groups, and each wave
// begins its sums with its rows' low-rank part, while the first tiles of the
// shared operands are on their way.  B_g m_i is summed
// by the matrix instructions of the layer's type: each m is split into two values
// of that type (three where fp32 outputs of bf16 values keep more), high and low
// part, whose products are as if the rank were two or three times as large.  For
// fp16 a row's m are first scaled by a power of two to less than 2 (8 at the end
// of 32 bits' range), which keeps them and their low parts in its range.  Infinite and
// zero m and factors give what they give unsplit: a finite m's parts are finite, the
// high part of one that is not zero is not zero, and only high parts meet infinities.
#include "grouped_device.hpp"

using namespace nerf_hip;
using namespace nerf_hip::grouped;

namespace {

// The power of two that scales values of at most `most` to less than 2 (8), and its
// inverse.  Beside an infinity the largest one: the sum is an infinity or NaN then, and
// what the finite values keep is that they are finite.
struct Power {
    float value, inverse;
};
__device__ __forceinline__ Power power_of(float most) {
    const uint32_t exponent = min(max(__float_as_uint(most) >> 23, 1u), 252u);
    if (most > 0.0f) return {__uint_as_float(exponent << 23), __uint_as_float((254u - exponent) << 23)};
    return {1.0f, 1.0f};
}
// What a value's first piece is rounded from (`scaled` by its row's power): one that is not
// zero stays so, as the smallest number of fp16 at least, and one that is finite too, as
// the largest of bf16 at most; the rest has the difference.
template <typename T>
__device__ __forceinline__ float to_round(float scaled, float value) {
    if constexpr (std::is_same_v<T, half_t>) return value != 0.0f && fabsf(scaled) < 0x1p-24f ? __builtin_copysignf(0x1p-24f, value) : scaled;
    return fabsf(value) < __builtin_inff() ? __builtin_amdgcn_fmed3f(value, -0x1.FEp127f, 0x1.FEp127f) : value;
}
// What a rounding leaves of a value: nothing of an infinity or NaN.
__device__ __forceinline__ float rest_of(float value, float rounded) { return fabsf(rounded) < __builtin_inff() ? value - rounded : 0.0f; }
// The factors of a value's pieces: all of them for the first piece (first[e] = 1),
// which has the value's sign; for the others, which may be zero or have the other
// sign, with zeros in place of infinities and NaN.  So an infinite factor gives what it
// gives with the value itself.
template <uint32_t kCount>
using u16s = unsigned short __attribute__((ext_vector_type(kCount)));
typedef u16s<8> u16x8;
template <typename T, typename V, typename First>
__device__ __forceinline__ V factors_of(V v, First first) {
    using Bits = u16s<sizeof(V) / 2u>;
    constexpr unsigned short kExponent = std::is_same_v<T, half_t> ? 0x7C00u : 0x7F80u;
    const Bits bits = __builtin_bit_cast(Bits, v), keep = (~bits & kExponent) | first;
    return __builtin_bit_cast(V, bits & (0 - __builtin_elementwise_min(keep, (Bits)1)));
}

// Whether any of the factors is an infinity or NaN.
template <typename T, typename V, uint32_t kCount>
__device__ __forceinline__ bool any_infinite(const V (&v)[kCount]) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    constexpr unsigned short kExponent = std::is_same_v<T, half_t> ? 0x7C00u : 0x7F80u;
    struct Words { uint32_t w[sizeof(V) / 4u]; };
    u16x2 most = {0, 0};
#pragma unroll
    for (uint32_t i = 0; i < kCount; ++i) {
        const Words words = __builtin_bit_cast(Words, v[i]);
#pragma unroll
        for (uint32_t j = 0; j < sizeof(V) / 4u; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, words.w[j] & 0x7FFF7FFFu));
    }
    return most[0] >= kExponent || most[1] >= kExponent;
}

// The low-rank part of a wave's sums: low [rows][rank] times wide, which is
// [groups][np][rank] (kPT: [groups][rank][np]).
template <typename T, bool kPT>
struct LowRank {
    static constexpr bool kOn = true;
    using x8 = typename Vec<T>::x8;
    const float* low;
    const T* wide;
    const float* scales;
    Groups G;
    uint32_t np, rank, pieces;
    bool vec_low, vec_wide;  // rows of low / of wide in whole aligned chunks

    // Eight of a row's values from r0, zeros beyond the rank.  Every load is made, from
    // inside the arrays, and what does not count is dropped: a branch would have them
    // wait for each other.
    __device__ __forceinline__ floatx8 low_eight(uint32_t position, uint32_t r0) const {
        const float* at = low + (uint64_t)min(position, G.rows - 1u) * rank;
        const bool none = r0 >= rank;
        floatx8 v;
        if (vec_low) {
            const floatx4* from = reinterpret_cast<const floatx4*>(at + (none ? 0u : r0));
            v.lo = from[0];
            v.hi = from[1];
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) v[e] = at[min(r0 + e, rank - 1u)];
        }
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) v[e] = r0 + e < rank ? v[e] : 0.0f;
        return v;
    }
    // Eight of wide's values at p from r0; others of the array where those are outside.
    __device__ __forceinline__ x8 wide_eight(uint32_t g, uint32_t p, uint32_t r0) const {
        const uint32_t column = min(p, np - 1u);
        x8 v;
        if constexpr (!kPT) {
            const T* at = wide + ((uint64_t)g * np + column) * rank;
            if (vec_wide) {
                v = *reinterpret_cast<const x8*>(at + (r0 < rank ? r0 : 0u));
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) v[e] = at[min(r0 + e, rank - 1u)];
            }
        } else {
            const T* at = wide + (uint64_t)g * rank * np + column;
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) v[e] = at[(uint64_t)min(r0 + e, rank - 1u) * np];
        }
        return v;
    }
    // Piece `piece` of eight values, scaled by their row's power.
    static __device__ __forceinline__ x8 piece_of(floatx8 v, float inverse, uint32_t piece) {
        floatx8 first;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) first[e] = to_round<T>(v[e] * inverse, v[e]);
        v *= inverse;
        x8 h = __builtin_convertvector(first, x8);
        for (uint32_t i = 0; i < piece; ++i) {
            const floatx8 back = __builtin_convertvector(h, floatx8);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) v[e] = rest_of(v[e], back[e]);
            h = __builtin_convertvector(v, x8);
        }
        return h;
    }

    // The group of position q0 + lane, of `count` positions: that of q0, and one more
    // for every offset up to the position.
    // asked: ask_offset()'s, the lane's offset where there are as many lanes.
    __device__ __forceinline__ uint32_t ask_offset() const {
        const uint32_t lane = threadIdx.x & 63u;
        return G.count < 64u && lane <= G.count ? G.offset(lane) : kNoRow;
    }
    __device__ __forceinline__ uint32_t group_of_lane(uint32_t asked, uint32_t q0, uint32_t count) const {
        const uint32_t lane = threadIdx.x & 63u, q_last = q0 + count - 1u;
        uint32_t mine;
        if (G.count < 64u) {
            const uint32_t offset = asked;
            const uint32_t before = (uint32_t)__popcll(__ballot(lane < G.count && offset <= q0)), end = (uint32_t)__popcll(__ballot(offset <= q_last));
            mine = before;
            for (uint32_t c = before; c < end; ++c) mine += (uint32_t)__builtin_amdgcn_readlane((int)offset, (int)c) <= q0 + lane;
        } else {
            const uint32_t before = count_at_most(G.count, q0, [&](uint32_t g) { return G.offset(g); });
            mine = before;
            for (uint32_t first = before; first <= G.count; first += 64u) {
                const uint32_t offset = first + lane <= G.count ? G.offset(first + lane) : kNoRow;
                const uint32_t some = (uint32_t)__popcll(__ballot(offset <= q_last));
                for (uint32_t c = 0; c < some; ++c) mine += (uint32_t)__builtin_amdgcn_readlane((int)offset, (int)c) <= q0 + lane;
                if (some < 64u) break;
            }
        }
        return lane < count && q0 + lane < G.rows && mine != 0u && mine <= G.count ? mine - 1u : kNoRow;
    }

    // Values of kFQ rows a lane for step `s` of 32 k, k counted as (piece, rank): a
    // quarter of the wave has eight of one piece.
    struct Step {
        uint32_t piece, r0;
    };
    // Which of wide's eight values a step takes as they are: those of first pieces within
    // the rank.  Of the others, m's are zeros or low pieces, factors_of() the finite ones.
    __device__ __forceinline__ u16x8 as_they_are(const Step& step) const {
        u16x8 first;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) first[e] = step.piece == 0u && step.r0 + e < rank;
        return first;
    }
    __device__ __forceinline__ Step step_of(uint32_t s) const {
        const uint32_t chunks = (rank + 7u) / 8u, chunk = 4u * s + ((threadIdx.x & 63u) >> 4), piece = chunk / chunks;
        return {piece < pieces ? piece : 0u, piece < pieces ? 8u * (chunk - piece * chunks) : rank};
    }
    __device__ __forceinline__ uint32_t steps() const { return (pieces * ((rank + 7u) / 8u) + 3u) / 4u; }
    template <uint32_t kFQ>
    __device__ __forceinline__ void fetch(floatx8 (&values)[kFQ], uint32_t q0, uint32_t s) const {
#pragma unroll
        for (uint32_t j = 0; j < kFQ; ++j) values[j] = low_eight(q0 + 16u * j + (threadIdx.x & 15u), step_of(s).r0);
    }
    // The power of two of the row of position q0 + lane.
    __device__ __forceinline__ Power power_of_lane(uint32_t q0) const {
        if constexpr (!std::is_same_v<T, half_t>) return {1.0f, 1.0f};
        const float* at = low + (uint64_t)min(q0 + (threadIdx.x & 63u), G.rows - 1u) * rank;
        float most = 0.0f;
        if (vec_low) {
            for (uint32_t r = 0; r < rank; r += 8u) {
                const floatx4 v = *reinterpret_cast<const floatx4*>(at + r), w = *reinterpret_cast<const floatx4*>(at + r + 4u);
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) most = fmaxf(most, fmaxf(fabsf(v[e]), fabsf(w[e])));
            }
        } else {
#pragma unroll 4
            for (uint32_t r = 0; r < rank; ++r) most = fmaxf(most, fabsf(at[r]));
        }
        return power_of(most);
    }
    // What position 16 j + lane % 16 has of a value that lane 16 j + lane % 16 holds.
    static __device__ __forceinline__ float of_row(float v, uint32_t j) { return std::is_same_v<T, half_t> ? __shfl(v, (int)(16u * j + (threadIdx.x & 15u))) : 1.0f; }
    // acc[i][j] of group g's rows += factor times the product of one step.  Rows of
    // other groups keep theirs, whatever this group's weights hold.
    template <uint32_t kFP, uint32_t kFQ, uint32_t kSome>
    __device__ __forceinline__ void add_group(floatx4 (&acc)[kFP][kFQ], uint32_t from, const x8 (&fp)[kSome], const x8 (&fq)[kFQ], uint64_t those, float power, float scale) const {
#pragma unroll
        for (uint32_t j = 0; j < kFQ; ++j) {
            const uint32_t rows = (uint32_t)(those >> (16u * j)) & 0xFFFFu;
            if (rows == 0u) continue;
            const float factor = of_row(power, j) * scale;
            const bool member  = rows >> (threadIdx.x & 15u) & 1u;
#pragma unroll
            for (uint32_t i = 0; i < kSome; ++i) {
                const floatx4 part = Vec<T>::mfma(fp[i], fq[j], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (uint32_t r = 0; r < 4u; ++r) acc[from + i][j][r] = member ? acc[from + i][j][r] + factor * part[r] : acc[from + i][j][r];
            }
        }
    }

    // acc[i][j]: 16 outputs from p0 + 16 i at 16 positions from q0 + 16 j, four
    // consecutive outputs of position lane % 16 a lane; zeros before.
    template <uint32_t kFP, uint32_t kFQ>
    __device__ __forceinline__ void begin(floatx4 (&acc)[kFP][kFQ], uint32_t p0, uint32_t q0) const {
        static_assert(16u * kFQ <= 64u);
        // The widest tiles' sums leave few registers: values are fetched as they are used.
        constexpr bool kTight = kFP * kFQ >= 32u;
        floatx8 values[kFQ];
        if (!kTight) fetch(values, q0, 0u);
        const uint32_t mine = group_of_lane(ask_offset(), q0, 16u * kFQ);
        if (__ballot(mine != kNoRow) == 0ull) return;
        const Power power = power_of_lane(q0);
        for (uint32_t s = 0; s < steps(); ++s) {
            const Step step = step_of(s);
            const u16x8 first = as_they_are(step);
            x8 fq[kFQ];
            if (kTight) fetch(values, q0, s);
#pragma unroll
            for (uint32_t j = 0; j < kFQ; ++j) fq[j] = piece_of(values[j], of_row(power.inverse, j), step.piece);
            if (!kTight && s + 1u < steps()) fetch(values, q0, s + 1u);
            // The groups of the wave's rows, one after another.
            for (uint64_t left = __ballot(mine != kNoRow); left;) {
                const uint32_t g = (uint32_t)__builtin_amdgcn_readlane((int)mine, __builtin_ctzll(left));
                const uint64_t those = __ballot(mine == g);
                left &= ~those;
                const float scale = scales ? scales[g] : 1.0f;
                // A few at a time in the widest tiles (8192 rows, rank 64, gradients of 4096 ->
                // 2048: 305 us with four, 325 with all eight, some of them spilled).
                constexpr uint32_t kSome = kTight ? 4u : kFP;
#pragma unroll
                for (uint32_t from = 0; from < kFP; from += kSome) {
                    x8 fp[kSome];
#pragma unroll
                    for (uint32_t i = 0; i < kSome; ++i) fp[i] = wide_eight(g, p0 + 16u * (from + i) + (threadIdx.x & 15u), step.r0);
#pragma unroll
                    for (uint32_t i = 0; i < kSome; ++i) fp[i] = factors_of<T>(fp[i], first);
                    add_group(acc, from, fp, fq, those, power.value, scale);
                }
            }
        }
    }

    // The same by several waves that add to the same sums, each its share of the
    // groups, in two parts: what is asked for first (the first step of the wave's
    // first groups) and what is added last.
    static constexpr uint32_t kAsked = 4u;
    template <uint32_t kFP, uint32_t kFQ>
    struct Asked {
        uint32_t offset, mine;
        floatx8 values[kFQ];
        Power power;
        x8 fp[kAsked][kFP];
        float scale[kAsked];
    };
    // The wave's groups: turn(number among them, group, its rows).
    template <typename Turn>
    __device__ __forceinline__ void for_groups(uint32_t mine, uint32_t share, uint32_t shares, Turn turn) const {
        uint32_t number = 0u, of_wave = 0u;
        for (uint64_t left = __ballot(mine != kNoRow); left; ++number) {
            const uint32_t g = (uint32_t)__builtin_amdgcn_readlane((int)mine, __builtin_ctzll(left));
            const uint64_t those = __ballot(mine == g);
            left &= ~those;
            if (number % shares == share) turn(of_wave++, g, those);
        }
    }
    template <uint32_t kFP, uint32_t kFQ>
    __device__ __forceinline__ Asked<kFP, kFQ> ask(uint32_t q0) const {
        Asked<kFP, kFQ> a;
        a.offset = ask_offset();
        fetch(a.values, q0, 0u);
        a.power = power_of_lane(q0);
        return a;
    }
    template <uint32_t kFP, uint32_t kFQ>
    __device__ __forceinline__ void ask_more(Asked<kFP, kFQ>& a, uint32_t p0, uint32_t q0, uint32_t share, uint32_t shares) const {
        a.mine = group_of_lane(a.offset, q0, 16u * kFQ);
        const Step step = step_of(0u);
        for_groups(a.mine, share, shares, [&](uint32_t n, uint32_t g, uint64_t) {
#pragma unroll
            for (uint32_t t = 0; t < kAsked; ++t)
                if (n == t) {
                    a.scale[t] = scales ? scales[g] : 1.0f;
#pragma unroll
                    for (uint32_t i = 0; i < kFP; ++i) a.fp[t][i] = wide_eight(g, p0 + 16u * i + (threadIdx.x & 15u), step.r0);
                }
        });
    }
    template <uint32_t kFP, uint32_t kFQ>
    __device__ __forceinline__ void add(floatx4 (&acc)[kFP][kFQ], const Asked<kFP, kFQ>& a, uint32_t p0, uint32_t q0, uint32_t share, uint32_t shares) const {
        if (__ballot(a.mine != kNoRow) == 0ull) return;
        for (uint32_t s = 0; s < steps(); ++s) {
            const Step step = step_of(s);
            const u16x8 first = as_they_are(step);
            floatx8 values[kFQ];
            x8 fq[kFQ];
            if (s) fetch(values, q0, s);
#pragma unroll
            for (uint32_t j = 0; j < kFQ; ++j) fq[j] = piece_of(s ? values[j] : a.values[j], of_row(a.power.inverse, j), step.piece);
            for_groups(a.mine, share, shares, [&](uint32_t n, uint32_t g, uint64_t those) {
                x8 fp[kFP];
                float scale;
                if (s == 0u && n < kAsked) {
#pragma unroll
                    for (uint32_t t = 0; t < kAsked; ++t)
                        if (n == t) {
                            scale = a.scale[t];
#pragma unroll
                            for (uint32_t i = 0; i < kFP; ++i) fp[i] = a.fp[t][i];
                        }
                } else {
                    scale = scales ? scales[g] : 1.0f;
#pragma unroll
                    for (uint32_t i = 0; i < kFP; ++i) fp[i] = wide_eight(g, p0 + 16u * i + (threadIdx.x & 15u), step.r0);
                }
#pragma unroll
                for (uint32_t i = 0; i < kFP; ++i) fp[i] = factors_of<T>(fp[i], first);
                add_group(acc, 0u, fp, fq, those, a.power.value, scale);
            });
        }
    }
};

// The shared product in tiles, see product().  8192 rows in 8 groups, rank 64, 2048 ->
// 4096 bf16 (the input gradient of a layer 4096 -> 2048) take 230 us, the same without
// adapters 170: what is added is the wait for the adapter's values at a tile's
// start, once a group in it, which nothing hides with one tile a CU.  (A copy of down
// with the ranks in a row, one load for eight, took as long.)
// As many waves a SIMD as LDS holds: with three registers more than they leave, odd
// rows' tiles of 128 ran one at a time (8192 rows of 1023 -> 2047, 214 us, so 138).
template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, uint32_t kDepth, bool kPT, Mode kMode, bool kGather, typename Out>
__global__ __launch_bounds__(kWP * kWQ * 64u, kBP > 64u || kMode == kDirect ? 2u : 4u) void k_adapter(GatheredOperands A, Out out, LowRank<T, kPT> more) {
    __shared__ uint32_t rows[kBQ];
    const uint32_t block = block_number(), tiles = A.tiles_p * A.tiles_q;
    if (block >= tiles) return;
    const uint32_t t = chip_tile(block, tiles), band = A.tiles_p > 4u ? 4u : 1u;
    const uint32_t first = t / (band * A.tiles_p) * band, high = min(band, A.tiles_q - first), in_band = t - first * A.tiles_p;
    const Place at{in_band / high * kBP, (first + in_band % high) * kBQ, 0u, A.nk, 0u, 0u};
    find_rows<kBQ>(out, rows, at.q0, A.nq);
    product<T, kBP, kBQ, kWP, kWQ, kDepth, kPT, false, kMode, kGather>(A, out, at, more);
}

// The same with few tiles: the waves share the groups.  32 rows in 32 groups, rank
// 16, 4096 -> 4096 bf16: 21 us and 9 for m, the layer without adapters 18; bound by the
// reading of 33 MB of weights in one round of workgroups (8 at a copy's rate).
template <typename T, uint32_t kFP, uint32_t kFQ, bool kPT, bool kWhole, typename Out>
__global__ __launch_bounds__(kFewWaves * 64u) void k_adapter_few(GatheredOperands A, Out out, LowRank<T, kPT> more) {
    __shared__ floatx4 lds[few_lds(kFP, kFQ) / 16u];
    __shared__ uint32_t rows[16u * kFQ];
    const Place at{blockIdx.x % A.tiles_p * 16u * kFP, blockIdx.x / A.tiles_p * 16u * kFQ, 0u, A.nk, 0u, 0u};
    few_tile<T, kFP, kFQ, kPT, false, !kWhole, true, kWhole>(A, out, at, reinterpret_cast<char*>(lds), nullptr, rows, more);
}

// Many rows, at most 32 kKS <= 256 k and 16 kRB <= 64 ranks, whole chunks: both
// low-rank products and the shared one in one pass over the rows, with the shared
// weights in registers (as k_stream in linear.hip) and the group's adapter in LDS.
// A wave computes its rows' m, 16 ranks at a time, from the same registers as the
// shared product (the waves of a row that hold other p do so again); lane 16 g + l
// ends with ranks 4 g .. 4 g + 3 of row l, and their high and low parts are what it
// has to hold for the next product, if that counts its k as (g, part, rank): no
// value moves between lanes.  A workgroup has consecutive positions, group by group.
// 262144 rows in 16 groups, rank 16, 256 -> 256 fp16, residual and pre: 140-145 us,
// 3.9 TB/s (tiles after a pass for m 206); its input gradient 156.
struct StreamRanks {
    const void* shrink;  // down [groups][rank][nk]; kPT: up [groups][nk][rank]
    float* low;          // m
    const uint32_t* index;  // of the outputs
    uint32_t count;
};
template <typename T, uint32_t kKS, uint32_t kRB, bool kPT, typename Out>
__global__ __launch_bounds__(kStreamWaves * 64u) void k_adapter_stream(GatheredOperands A, Out out, LowRank<T, kPT> more, StreamRanks R, uint32_t p_waves) {
    out.vec = true;
    constexpr uint32_t kThreads = kStreamWaves * 64u, kFP = 4u, kSP = 16u * kFP, kBP = 256u, kLanes = kSP / 8u, kPasses = 16u * kLanes / 64u;
    using x8 = typename Vec<T>::x8;
    typedef T x4 __attribute__((ext_vector_type(4)));
    __shared__ uint4 lds[kBP * 8u];
    __shared__ floatx4 lds_bias[Out::kBias ? kBP / 4u : 1u];
    __shared__ uint32_t x_rows[kStreamChunk], y_rows[kStreamChunk];
    __shared__ x8 lds_shrink[kRB * kKS * 64u];
    __shared__ x8 lds_grow[kRB * kBP * 4u];  // factors of high parts, then of low ones
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, l = lane & 15u, quarter = lane >> 4;
    const uint32_t wp = wave % p_waves * kSP, p0 = blockIdx.y * p_waves * kSP, waves_q = kStreamWaves / p_waves;
    const Groups& G = more.G;

    x8 fp[kKS][kFP];
    hold_weights<T, kBP, kPT>(A, out, p0, wp, lds, lds_bias, fp);

    const uint32_t row = lane / kLanes, col = 8u * (lane % kLanes), p = p0 + wp + col;
    const uint32_t n = p < A.np ? min(8u, A.np - p) : 0u;
    floatx4* strip = reinterpret_cast<floatx4*>(lds) + wave * (kSP * 4u);
    constexpr bool kLate = sizeof(typename Out::Aux) > 16u;
    const uint32_t each = (A.nq + 16u * gridDim.x - 1u) / (16u * gridDim.x) * 16u;
    const uint64_t from = (uint64_t)chip_tile(blockIdx.x, gridDim.x) * each;
    const uint32_t last = (uint32_t)min((uint64_t)A.nq, from + each);
    const bool keeps_low = wp == 0u && blockIdx.y == 0u;
    for (uint32_t pos = (uint32_t)min(from, (uint64_t)last), part_end; pos < last; pos = part_end) {
        // The group of the next positions, or none, and where its part of them ends.
        const uint32_t c = __builtin_amdgcn_readfirstlane(count_at_most(G.count, pos, [&](uint32_t g) { return G.offset(g); }));
        const uint32_t group_end = c ? G.offset(c) : 0u, g = c ? c - 1u : 0u;
        const bool member = pos < group_end;
        const uint32_t limit = member ? group_end : c < G.count ? G.offset(c) : A.nq;
        part_end = min(min(limit > pos ? limit : A.nq, last), pos + kStreamChunk);
        const uint32_t end = part_end, tiles = (end - pos + 15u) / 16u;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < end - pos; i += kThreads) {
            x_rows[i] = gathered_row(A.q_index, A.q_count, pos + i, end);
            y_rows[i] = R.index ? gathered_row(R.index, R.count, pos + i, end) : i;
        }
        if (member) {
            const T* shrink = (const T*)R.shrink;
            for (uint32_t i = threadIdx.x; i < kRB * kKS * 64u; i += kThreads) {
                const uint32_t r = i / (kKS * 64u) * 16u + i % 16u, k = i / 64u % kKS * 32u + i / 16u % 4u * 8u;
                const bool inner = r < more.rank && k < A.nk;
                x8 v;
                if constexpr (!kPT) {
                    v = *reinterpret_cast<const x8*>(shrink + (inner ? ((uint64_t)g * more.rank + r) * A.nk + k : 0ull));
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) v[e] = shrink[inner ? ((uint64_t)g * A.nk + k + e) * more.rank + r : 0ull];
                }
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) v[e] = inner ? v[e] : (T)0.0f;
                lds_shrink[i] = v;
            }
            for (uint32_t i = threadIdx.x; i < kRB * kBP * 4u; i += kThreads) {
                const uint32_t r = i / (kBP * 4u) * 16u + i / 16u % 4u * 4u, at = p0 + i / 64u % (kBP / 16u) * 16u + i % 16u;
                x4 v;
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) {
                    const bool inner = at < A.np && r + e < more.rank;
                    const T w = more.wide[!inner ? 0ull : kPT ? ((uint64_t)g * more.rank + r + e) * A.np + at : ((uint64_t)g * A.np + at) * more.rank + r + e];
                    v[e] = inner ? w : (T)0.0f;
                }
                lds_grow[i] = __builtin_shufflevector(v, factors_of<T>(v, u16s<4>{0, 0, 0, 0}), 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
        const float scale = member && more.scales ? more.scales[g] : 1.0f;
        __syncthreads();

        struct Coming {
            uint4 q[kKS];
            uint32_t none;
            typename Out::Aux aux[kPasses];
        } c0;
        const uint32_t q0 = R.index ? 0u : pos;
        auto row_of       = [&](uint32_t tile, uint32_t pass) {
            const uint32_t r = tile * 16u + (64u / kLanes) * pass + row;
            return r < end - pos ? y_rows[r] : kNoRow;
        };
        auto fetch_q = [&](uint32_t tile) {
            const uint32_t r = x_rows[min(tile * 16u + l, end - pos - 1u)];
            c0.none          = r == kNoRow;
            const T* at      = (const T*)A.q + (uint64_t)(r == kNoRow ? 0u : r) * A.ldq + 8u * quarter;
#pragma unroll
            for (uint32_t s = 0; s < kKS; ++s)
                if (32u * s < A.nk) c0.q[s] = *reinterpret_cast<const uint4*>(at + 32u * s);
        };
        auto fetch_aux = [&](uint32_t tile, uint32_t t) {
            const uint32_t r = row_of(tile, t);
            c0.aux[t]        = out.load(q0, r, p, r != kNoRow ? n : 0u);
        };
#pragma unroll
        for (uint32_t s = 0; s < kKS; ++s) c0.q[s] = uint4{0u, 0u, 0u, 0u};
        const uint32_t first_tile = __builtin_amdgcn_readfirstlane(wave / p_waves);
        if (first_tile < tiles) {
            fetch_q(first_tile);
#pragma unroll
            for (uint32_t t = 0; t < kPasses; ++t) fetch_aux(first_tile, t);
        }
        for (uint32_t tile = first_tile; tile < tiles; tile += waves_q) {
            const uint32_t later = tile + waves_q;
            if (c0.none) {
#pragma unroll
                for (uint32_t s = 0; s < kKS; ++s) c0.q[s] = uint4{0u, 0u, 0u, 0u};
            }
            floatx4 acc[kFP];
#pragma unroll
            for (uint32_t i = 0; i < kFP; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            if (member) {
#pragma unroll
                for (uint32_t rb = 0; rb < kRB; ++rb) {
                    floatx4 m = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (uint32_t s = 0; s < kKS; ++s) m = Vec<T>::mfma(lds_shrink[(rb * kKS + s) * 64u + lane], __builtin_bit_cast(x8, c0.q[s]), m);
                    if constexpr (kPT) m *= scale;
                    const uint32_t position = pos + tile * 16u + l, r = 16u * rb + 4u * quarter;
                    // Beyond the rank: an infinite input makes NaN of the zeros there.
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) m[e] = r + e < more.rank ? m[e] : 0.0f;
                    if (keeps_low && position < end) {
                        float* to = R.low + (uint64_t)position * more.rank + r;
                        if (more.vec_low) {
                            if (r < more.rank) *reinterpret_cast<floatx4*>(to) = m;
                        } else {
#pragma unroll
                            for (uint32_t e = 0; e < 4u; ++e)
                                if (r + e < more.rank) to[e] = m[e];
                        }
                    }
                    float factor = kPT ? 1.0f : scale;
                    floatx4 first;
                    if constexpr (std::is_same_v<T, half_t>) {
                        float most = fmaxf(fmaxf(fabsf(m[0]), fabsf(m[1])), fmaxf(fabsf(m[2]), fabsf(m[3])));
                        most = fmaxf(most, __shfl_xor(most, 16));
                        most = fmaxf(most, __shfl_xor(most, 32));
                        const Power power = power_of(most);
#pragma unroll
                        for (uint32_t e = 0; e < 4u; ++e) first[e] = to_round<T>(m[e] * power.inverse, m[e]);
                        m *= power.inverse;
                        factor *= power.value;
                    } else {
#pragma unroll
                        for (uint32_t e = 0; e < 4u; ++e) first[e] = to_round<T>(m[e], m[e]);
                    }
                    const x4 high = __builtin_convertvector(first, x4);
                    floatx8 rest;
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) rest[e] = e < 4u ? first[e] : rest_of(m[e - 4u], (float)high[e - 4u]);
                    const x8 pieces = __builtin_convertvector(rest, x8);
                    x8 third;
                    if (more.pieces == 3u) {
#pragma unroll
                        for (uint32_t e = 0; e < 8u; ++e) third[e] = e < 4u ? (T)0.0f : (T)rest_of(rest[e], (float)pieces[e]);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < kFP; ++i) {
                        const x8 w = lds_grow[(rb * (kBP / 16u) + wp / 16u + i) * 64u + lane];
                        floatx4 part = Vec<T>::mfma(w, pieces, floatx4{0.0f, 0.0f, 0.0f, 0.0f});
                        if (more.pieces == 3u) part = Vec<T>::mfma(__builtin_shufflevector(w, w, 4, 5, 6, 7, 4, 5, 6, 7), third, part);
                        acc[i] += factor * part;
                    }
                }
            }
#pragma unroll
            for (uint32_t s = 0; s < kKS; ++s)
#pragma unroll
                for (uint32_t i = 0; i < kFP; ++i) acc[i] = Vec<T>::mfma(fp[s][i], __builtin_bit_cast(x8, c0.q[s]), acc[i]);
            typename Out::Aux aux[kPasses];
#pragma unroll
            for (uint32_t t = 0; t < kPasses; ++t) aux[t] = c0.aux[t];
            if (later < tiles) {
                fetch_q(later);
#pragma unroll
                for (uint32_t t = 0; t < kPasses; ++t)
                    if (!kLate) fetch_aux(later, t);
            }
#pragma unroll
            for (uint32_t i = 0; i < kFP; ++i) strip[l * (kSP / 4u) + ((4u * i + quarter) ^ (l & 7u))] = acc[i];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (uint32_t t = 0; t < kPasses; ++t) {
                const uint32_t r = (64u / kLanes) * t + row, to_row = row_of(tile, t);
                floatx8 v;
                v.lo = strip[r * (kSP / 4u) + ((col / 4u) ^ (r & 7u))];
                v.hi = strip[r * (kSP / 4u) + ((col / 4u + 1u) ^ (r & 7u))];
                out.put(q0, to_row, p, to_row != kNoRow ? n : 0u, v, bias8<Out>(reinterpret_cast<const float*>(lds_bias), wp + col), aux[t]);
                if (kLate) fetch_aux(later, t);
            }
            asm volatile("" ::: "memory");
        }
    }
}

// Operands of fewer than eight values in all: a thread an output of a position.
template <typename T, bool kPT, typename Out>
__global__ __launch_bounds__(64) void k_adapter_tiny(GatheredOperands A, Out out, LowRank<T, kPT> more) {
    __shared__ uint32_t rows[1];
    const Groups& G = more.G;
    for (uint32_t position = blockIdx.x; position < A.nq; position += gridDim.x) {
        Out mine = out;
        __syncthreads();
        find_rows<1u>(mine, rows, position, position + 1u);
        __syncthreads();
        const Part part     = part_at(G, 1u, position);
        const bool member   = part.q0 < part.end;
        const uint32_t g    = part.group, from = gathered_row(A.q_index, A.q_count, position, position + 1u);
        const float scale   = member && more.scales ? more.scales[g] : 1.0f;
        for (uint32_t p = 8u * threadIdx.x; p < A.np; p += 512u) {
            const uint32_t n = min(8u, A.np - p);
            const typename Out::Aux aux = mine.load(position, 0u, p, n);
            floatx8 v = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, b = v;
            for (uint32_t k = 0; k < A.nk; ++k) {
                const float x = from == kNoRow ? 0.0f : (float)((const T*)A.q)[from * A.ldq + k];
#pragma unroll
                for (uint32_t r = 0; r < 8u; ++r)
                    if (r < n) v[r] += x * (float)((const T*)A.p)[kPT ? k * A.ldp + p + r : (p + r) * A.ldp + k];
            }
            for (uint32_t k = 0; member && k < more.rank; ++k) {
                const float m = scale * more.low[(uint64_t)position * more.rank + k];
#pragma unroll
                for (uint32_t r = 0; r < 8u; ++r)
                    if (r < n) v[r] += m * (float)more.wide[kPT ? ((uint64_t)g * more.rank + k) * A.np + p + r : ((uint64_t)g * A.np + p + r) * more.rank + k];
            }
            if constexpr (Out::kBias) {
                if (mine.bias) {
#pragma unroll
                    for (uint32_t r = 0; r < 8u; ++r)
                        if (r < n) b[r] = mine.bias[p + r];
                }
            }
            mine.put(position, 0u, p, n, v, b, aux);
        }
    }
}

// ------------------------------------------------------- gradients of adapters
// out_g(w, r) = scale_g sum_i wide(i, w) low(i, r): wide 16-bit rows, as an index
// names them, low 32-bit by position; kBW wide x kBR low values a workgroup, sums
// over parts of `size` positions of a group.  out is [groups][nw][nr], or with
// `low_major` [groups][nr][nw].
// For bf16 each low value is split into three of that type (24 bits; below 2^-110
// their last ones are lost), whose products take three sixteenths of the
// 32-bit instruction's time.  fp16 values would need a scale a row for that, which a
// sum over rows cannot take out again: the 32-bit instruction, four positions at a
// time.  8192 rows in 8 groups, rank 64, 4096 values: 46 us in bf16 (by the 32-bit
// instruction, each wave with all of r, 72; split so, 63; one wave for 16 of r, as it
// is now, reads and splits a value once), 2048 values 30.  What is left is the waits for
// gathered rows, two loads after each other, in parts of a few tiles; memory
// alone would take 13.  262144 rows, rank 16, 256 values, fp16: 45 us, 3.3 TB/s.
struct RankSums {
    const void* wide;
    const float* low;
    const float* scales;
    float *out, *parts;
    const uint32_t* index;
    uint64_t ld;
    uint32_t count, nw, nr, tiles_w, tiles_r;
    bool low_major;
};
constexpr uint32_t kBW = 128u;

// Tile of 64 positions x kBR low values straight into LDS, for rows that are whole
// multiples of 16 bytes; zeros outside.
template <uint32_t kBR>
struct LowLoader {
    static constexpr uint32_t kLoads = kBK * kBR / 4u / 256u;
    const float* base;
    uint32_t step;

    __device__ __forceinline__ void begin(const float* low, uint32_t nr, uint32_t r0, uint32_t k0) {
        base = low + (uint64_t)k0 * nr + r0;
        step = kBK * nr;
    }
    __device__ __forceinline__ void issue(float* lds, uint32_t nr, uint32_t r0, int left) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)0x7FFFFFFF, 0x00020000);
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t s = i * 256u + threadIdx.x, line = s / (kBR / 4u), r = s % (kBR / 4u) * 4u;
            const uint32_t at = (int)line < left && r0 + r < nr ? (line * nr + r) * 4u : kBeyond;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + (i * 256u + wave * 64u) * 4u), 16, (int)at, 0, 0, 0);
        }
        base += step;
    }
};

// kMode kDirect: both operands straight into LDS, the next tile's on their way;
// else through registers, at any alignment.
template <typename T, uint32_t kBR, Mode kMode, bool kGather>
__global__ __launch_bounds__(256) void k_rank_sums(RankSums A, Groups G, uint32_t size, uint32_t most) {
    // Waves side by side in r first, so that a low value is read and split by as few as
    // can be.
    constexpr uint32_t kWR = kBR / 16u, kFW = 2u * kWR;
    __shared__ uint4 wide0[kBW * 8u], wide1[kMode == kDirect ? kBW * 8u : 1u];
    __shared__ float low0[kBK * kBR], low1[kMode == kDirect ? kBK * kBR : 1u];
    const uint32_t tiles = A.tiles_w * A.tiles_r, t = dealt_tile(block_number(), most, tiles);
    if (t >= most * tiles) return;
    const Part part = part_of(G, size, t / tiles);
    if (part.q0 >= part.end && part.number) return;
    const uint32_t w0 = t % tiles % A.tiles_w * kBW, r0 = t % tiles / A.tiles_w * kBR;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, l = lane & 15u, quarter = lane >> 4;
    const uint32_t end = min(part.end, part.q0 + size);
    const uint32_t wave_w = wave / kWR * 16u * kFW, wave_r = wave % kWR * 16u;
    floatx4 acc[kFW];
#pragma unroll
    for (uint32_t i = 0; i < kFW; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t base = fragment_base<kBW, true>(wave_w);
    auto multiply = [&](const uint4* wide, const float* low) {
#pragma unroll
        for (uint32_t step = 0; step < 2u; ++step) {
            typename Vec<T>::x8 w[kFW];
#pragma unroll
            for (uint32_t i = 0; i < kFW; ++i) {
                w[i] = fragment<T, kBW, true>(wide, base, i, step);
                settle_here(w[i]);
            }
            floatx8 m;
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) m[e] = low[(32u * step + 8u * quarter + e) * kBR + wave_r + l];
            if constexpr (std::is_same_v<T, bf16_t>) {
#pragma unroll
                for (uint32_t piece = 0; piece < 3u; ++piece) {
                    // The first one towards zero, so that a finite value's is finite: the two
                    // others hold the 16 bits that are left.
                    floatx8 first = m;
                    if (piece == 0u) {
#pragma unroll
                        for (uint32_t e = 0; e < 8u; ++e) first[e] = __uint_as_float(__float_as_uint(m[e]) & 0xFFFF0000u);
                    }
                    const typename Vec<T>::x8 h = __builtin_convertvector(first, typename Vec<T>::x8);
#pragma unroll
                    for (uint32_t i = 0; i < kFW; ++i) acc[i] = Vec<T>::mfma(w[i], h, acc[i]);
                    const floatx8 back = piece == 0u ? first : __builtin_convertvector(h, floatx8);
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) m[e] = rest_of(m[e], back[e]);
                    // (For every step alike: 8192 rows of 4096 -> 2048, rank 64, 324 us, so 305.)
                    if (piece == 0u && __ballot(any_infinite<T>(w))) {
#pragma unroll
                        for (uint32_t i = 0; i < kFW; ++i) w[i] = factors_of<T>(w[i], (u16x8)0);
                    }
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kFW; ++i) {
                    const floatx8 v = __builtin_convertvector(w[i], floatx8);
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], m[e], acc[i], 0, 0, 0);
                }
            }
        }
    };
    if constexpr (kMode == kDirect) {
        std::conditional_t<kGather, GatherLoader<T, kBW, true, 256u>, Loader<T, kBW, true, 256u>> load;
        LowLoader<kBR> load_low;
        if constexpr (kGather) load.begin((const T*)A.wide, A.index, A.count, A.ld, A.nw, w0, part.q0, end);
        else load.begin((const T*)A.wide, A.ld, A.nw, w0, part.q0);
        load_low.begin(A.low, A.nr, r0, part.q0);
        auto issue = [&](uint4* wide, float* low, int left) {
            load_low.issue(low, A.nr, r0, left);
            if constexpr (kGather) load.issue(wide, left, A.index, A.count, A.ld, A.nw, w0);
            else load.issue(wide, left);
        };
        constexpr int kStep = (int)kBK;
        int left            = (int)(end - part.q0);
        if (left > 0) issue(wide0, low0, left);
        for (; left > 0; left -= 2 * kStep) {
            arrived<0u>();
            issue(wide1, low1, left - kStep);
            multiply(wide0, low0);
            arrived<0u>();
            if (left > 2 * kStep) issue(wide0, low0, left - 2 * kStep);
            multiply(wide1, low1);
        }
    } else {
        GatherStager<T, kBW, true, 256u> stage;
        stage.begin(A.index, A.count, part.q0, end);
        constexpr uint32_t kLow = kBK * kBR / 256u;
        float held[kLow];
        auto fetch = [&](uint32_t k) {
            stage.fetch((const T*)A.wide, A.index, A.count, A.ld, A.nw, w0, k, end);
#pragma unroll
            for (uint32_t i = 0; i < kLow; ++i) {
                const uint32_t e = i * 256u + threadIdx.x, line = k + e / kBR, r = r0 + e % kBR;
                held[i] = line < end && r < A.nr ? A.low[(uint64_t)line * A.nr + r] : 0.0f;
            }
        };
        if (part.q0 < end) fetch(part.q0);
        for (uint32_t k = part.q0; k < end; k += kBK) {
            stage.keep(wide0, (const T*)A.wide, A.ld, A.nw, w0, k, end);
#pragma unroll
            for (uint32_t i = 0; i < kLow; ++i) low0[i * 256u + threadIdx.x] = held[i];
            __syncthreads();
            if (k + kBK < end) fetch(k + kBK);
            multiply(wide0, low0);
            __syncthreads();
        }
    }
    const uint64_t length = (uint64_t)A.nw * A.nr;
    float* out = part.number ? A.parts + place_of(G, part, size) * length : A.out + part.group * length;
    const float scale = A.scales ? A.scales[part.group] : 1.0f;
    const uint32_t r = r0 + wave_r + l;
#pragma unroll
    for (uint32_t i = 0; i < kFW; ++i)
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
            const uint32_t w = w0 + wave_w + 16u * i + 4u * quarter + e;
            if (r < A.nr && w < A.nw) out[A.low_major ? (uint64_t)r * A.nw + w : (uint64_t)w * A.nr + r] = scale * acc[i][e];
        }
}

// Wide arrays of fewer than eight values in all: one thread an output.
template <typename T>
__global__ __launch_bounds__(256) void k_rank_tiny_sums(RankSums A, Groups G) {
    const uint64_t at = block_number() * 256ull + threadIdx.x, length = (uint64_t)A.nw * A.nr;
    if (at >= G.count * length) return;
    const uint32_t g = (uint32_t)(at / length), e = (uint32_t)(at % length), w = A.low_major ? e % A.nw : e / A.nr, r = A.low_major ? e / A.nw : e % A.nr;
    float v = 0.0f;
    for (uint32_t i = G.offset(g), end = G.offset(g + 1u); i < end; ++i) {
        const uint32_t row = gathered_row(A.index, A.count, i, end);
        v += (row == kNoRow ? 0.0f : (float)((const T*)A.wide)[row * A.ld + w]) * A.low[(uint64_t)i * A.nr + r];
    }
    A.out[at] = (A.scales ? A.scales[g] : 1.0f) * v;
}

// ------------------------------------------------------------------- host
template <typename T, bool kPT, typename Out>
hipError_t launch_adapter(GatheredOperands A, Out out, const LowRank<T, kPT>& more, hipStream_t stream) {
    const uint64_t weights = (uint64_t)A.np * A.nk, values = (uint64_t)(A.q_count - 1u) * A.ldq + A.nk;
    if (weights < 8u || values < 8u) {
        k_adapter_tiny<T, kPT, Out><<<std::min(A.nq, 64u * device_cu_count()), 64, 0, stream>>>(A, out, more);
        return hipGetLastError();
    }
    auto launch = [&](auto kernel, uint32_t bp, uint32_t bq, uint32_t threads) {
        A.tiles_p = ceil_div(A.np, bp);
        A.tiles_q = ceil_div(A.nq, bq);
        kernel<<<grid_of((uint64_t)A.tiles_p * A.tiles_q), threads, 0, stream>>>(A, out, more);
        return hipGetLastError();
    };
    const bool gather = A.q_index != nullptr;
    const bool words  = !whole_chunks(A.p, A.ldp, kPT ? A.np : A.nk) || !whole_chunks(A.q, A.ldq, A.nk) || (gather && !near(A.q_count, A.ldq));
    const uint64_t cus = device_cu_count();
    auto tiles_of      = [&](uint32_t p, uint32_t q) { return (uint64_t)ceil_div(A.np, p) * ceil_div(A.nq, q); };
    auto tiles         = [&](uint32_t b) { return tiles_of(b, b); };
    // us of a forward call, few of 16 x 16 / of 16 x 32 / of 32 x 32 / tiles of 64, bf16,
    // rank 16, 4096 -> 4096: 16 rows 24 / 25 / 28 / 33; 32 rows 35 / 30 / 32 / 38; 64 rows 56 /
    // 45 / 32 / 36; 128 rows 95 / 76 / 50 / 35; 1024 -> 1024: 64 rows 12 / 13 / 14 / 17, 128
    // rows 16 / 13 / 14 / 15, 512 rows 43 / 33 / 23 / 15.
    if (A.nk <= kFewMaxK) {
        auto few = [&](auto fp, auto fq) {
            const bool whole = A.nk % 32u == 0u && (!kPT || A.np % (16u * fp()) == 0u) && !odd_rows(A.p, A.ldp) && !odd_rows(A.q, A.ldq);
            if (whole) return launch(k_adapter_few<T, fp(), fq(), kPT, true, Out>, 16u * fp(), 16u * fq(), kFewWaves * 64u);
            return launch(k_adapter_few<T, fp(), fq(), kPT, false, Out>, 16u * fp(), 16u * fq(), kFewWaves * 64u);
        };
        using One = std::integral_constant<uint32_t, 1u>;
        using Two = std::integral_constant<uint32_t, 2u>;
        if (tiles(16u) <= cus) return few(One{}, One{});
        if (tiles_of(16u, 32u) <= cus) return few(One{}, Two{});
        if (tiles(32u) <= cus) return few(Two{}, Two{});
    }
    // us, tiles of 64 / of 128: 2048 -> 2048, 2048 rows (1024, 256 tiles) 44 / 39, 8192 rows
    // 150 / 97; 256 -> 256, 16384 rows (1024, 256) 20.7 / 20.2.  By words, one buffer and two
    // barriers a step: 255 -> 255, 16384 rows (256 of 128) 34 / 39, 32768 54 / 47, 1023 -> 1023,
    // 4096 rows (256) 57 / 64, 8192 109 / 93.
    const bool by_128 = A.np > 64u && A.nq > 64u && tiles(128u) >= (words ? 2u : 1u) * cus;
    if (words) return by_128 ? launch(k_adapter<T, 128, 128, 2, 2, 2, kPT, kByWords, true, Out>, 128u, 128u, 256u) : launch(k_adapter<T, 64, 64, 2, 2, 2, kPT, kByWords, true, Out>, 64u, 64u, 256u);
    // A tile of 256 takes a CU nearly as long as four of 128, so it needs full rounds: us of
    // a call, 128 / 256, 2048 -> 2048 rank 16, 4096 rows (1 round for 2) 54 / 81, 8192 (1 for
    // 4) 93-97 / 94-98; gradients of 4096 -> 2048, rank 64, 6144 rows (2 for 6) 265 / 291, 8192
    // (2 for 8) 338 / 319, 10240 (3 for 10) 404 / 417, 12288 rank 16 (3 for 12) 364 / 338;
    // 512 -> 512, 65536 rows (2 for 8) 85-90 / 89.
    if (A.np > 128u && A.nq > 128u && A.nk >= 1024u && 15u * ((tiles(256u) + cus - 1u) / cus) * cus <= 4u * tiles(128u))
        return gather ? launch(k_adapter<T, 256, 256, 2, 4, 2, kPT, kDirect, true, Out>, 256u, 256u, 512u) : launch(k_adapter<T, 256, 256, 2, 4, 2, kPT, kDirect, false, Out>, 256u, 256u, 512u);
    if (by_128) return gather ? launch(k_adapter<T, 128, 128, 2, 2, 2, kPT, kDirect, true, Out>, 128u, 128u, 256u) : launch(k_adapter<T, 128, 128, 2, 2, 2, kPT, kDirect, false, Out>, 128u, 128u, 256u);
    return gather ? launch(k_adapter<T, 64, 64, 2, 2, 4, kPT, kDirect, true, Out>, 64u, 64u, 256u) : launch(k_adapter<T, 64, 64, 2, 2, 4, kPT, kDirect, false, Out>, 64u, 64u, 256u);
}

// Whether k_adapter_stream takes a layer: with so many rows that its start, and the
// loading of an adapter at every group's first row, are small beside them.  Streamed /
// by tiles with the low-rank products before them, us, fp16, residual and pre (gradients:
// add, dx and both sums):
//   256 -> 256, rank 16: 65536 rows in 16 groups 50 / 56, in 256 60 / 60, in 1024 87 / 68;
//     131072 in 512 104 / 117, in 1024 120 / 120; 262144 in 16 146 / 206, in 1024 181 / 218,
//     in 4096 262 / 245; 32768 in 16 32 / 27.  Gradients 65536 in 16 89 / 104, in 256 104 /
//     111, in 1024 146 / 130; 262144 in 1024 298 / 364, in 4096 436 / 443.
//   Rank 32: 65536 in 64 65 / 72, in 256 79 / 75; 131072 in 256 120 / 139, in 1024 164 / 144;
//     262144 in 1024 233 / 264.
//   Less work a group is less to load: 64 -> 64, rank 64, 65536 in 256 45 / 57, rank 16 in
//     1024 44 / 36; 128 -> 128, rank 64, 65536 in 64 45 / 54, in 256 64 / 56.
// Four blocks of ranks for more than 128 k spill, and several waves compute the same m
// for more than 64 p: 256 -> 256, rank 64, 131072 rows in 1 group 173 / 173, in 64 183 / 176;
// 262144 in 64 325 / 338, in 256 353 / 346; gradients 65536 in 16 212 / 207, 131072 in 64
// 364 / 383, 262144 in 256 671 / 707, in 1024 747 / 722; 256 -> 128 65536 in 16 68 / 55, 262144
// 189 / 201.  Rank 48, which takes as long: 262144 in 16 316 / 275, gradients 598 / 603, 256
// -> 128 186 / 173.  256 -> 64, rank 64, 65536 in 16 52 / 54.
template <typename T, bool kPT>
bool streamed(const GatheredOperands& A, const LowRank<T, kPT>& more, const void* shrink, bool vec, const uint32_t* index, uint32_t count, uint64_t widest) {
    const uint32_t blocks = more.rank <= 16u ? 1u : more.rank <= 32u ? 2u : 4u;
    const bool spills     = blocks == 4u && A.nk > 128u && A.np > 64u;
    const uint64_t start  = !spills ? 32768u : kPT ? 98304u : 196608u, group = 48u + blocks * (A.nk + A.np) / 8u;
    if (A.nq < 65536u || A.nq < start + more.G.count * group || (spills && more.rank <= 48u)) return false;
    return A.nk <= 256u && A.nk % 32u == 0u && A.np <= 512u && more.rank <= 64u && vec && whole_chunks(A.p, A.ldp, kPT ? A.np : A.nk) && whole_chunks(A.q, A.ldq, A.nk) && aligned(shrink, 16u) && stream_outputs_near(index != nullptr, count, widest);
}

template <typename T, bool kPT, typename Out>
hipError_t launch_stream(const GatheredOperands& A, const Out& out, const LowRank<T, kPT>& more, const StreamRanks& R, hipStream_t stream) {
    uint32_t p_waves = 1u;
    while (p_waves < 4u && 64u * p_waves < A.np) p_waves *= 2u;
    const uint32_t across = ceil_div(A.np, 64u * p_waves);
    const dim3 grid(std::max(1u, device_cu_count() / across), across);
    auto launch = [&](auto steps, auto ranks) {
        k_adapter_stream<T, steps(), ranks(), kPT, Out><<<grid, kStreamWaves * 64u, 0, stream>>>(A, out, more, R, p_waves);
        return hipGetLastError();
    };
    auto by_rank = [&](auto steps) {
        if (more.rank <= 16u) return launch(steps, std::integral_constant<uint32_t, 1u>{});
        if (more.rank <= 32u) return launch(steps, std::integral_constant<uint32_t, 2u>{});
        return launch(steps, std::integral_constant<uint32_t, 4u>{});
    };
    if (A.nk <= 64u) return by_rank(std::integral_constant<uint32_t, 2u>{});
    if (A.nk <= 128u) return by_rank(std::integral_constant<uint32_t, 4u>{});
    return by_rank(std::integral_constant<uint32_t, 8u>{});
}

template <typename T>
hipError_t launch_rank_sums(RankSums A, const Groups& G, Workspace ws, hipStream_t stream) {
    const uint64_t length = (uint64_t)A.nw * A.nr;
    if (G.rows == 0u || (uint64_t)(A.count - 1u) * A.ld + A.nw < 8u) {
        k_rank_tiny_sums<T><<<grid_of((G.count * length + 255u) / 256u), 256, 0, stream>>>(A, G);
        return hipGetLastError();
    }
    // Parts enough for two workgroups a CU; one, four or eight: within 2 %.
    auto launch = [&](auto kernel, uint32_t br) {
        A.tiles_w = ceil_div(A.nw, kBW);
        A.tiles_r = ceil_div(A.nr, br);
        const uint64_t tiles = (uint64_t)A.tiles_w * A.tiles_r;
        const uint32_t size  = part_size(G.rows, tiles, 2u * device_cu_count(), 4u * length, ws.bytes), most = G.rows / size + G.count;
        A.parts              = ws.data;
        kernel<<<grid_of(dealt_blocks(most, (uint32_t)tiles)), 256, 0, stream>>>(A, G, size, most);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || size >= G.rows) return e;
        return launch_join(G, size, A.out, ws.data, length, nullptr, nullptr, 0u, stream);
    };
    auto by_rank = [&](auto mode, auto gather) {
        if (A.nr <= 16u) return launch(k_rank_sums<T, 16, mode(), gather()>, 16u);
        if (A.nr <= 32u) return launch(k_rank_sums<T, 32, mode(), gather()>, 32u);
        return launch(k_rank_sums<T, 64, mode(), gather()>, 64u);
    };
    using Direct = std::integral_constant<Mode, kDirect>;
    if (!whole_chunks(A.wide, A.ld, A.nw) || A.nr % 4u != 0u || !aligned(A.low, 16u) || (A.index && !near(A.count, A.ld))) return by_rank(std::integral_constant<Mode, kByWords>{}, std::true_type{});
    return A.index ? by_rank(Direct{}, std::true_type{}) : by_rank(Direct{}, std::false_type{});
}

template <typename T, bool kPT>
LowRank<T, kPT> low_rank(const float* low, const void* wide, const float* scales, const Groups& G, uint32_t np, uint32_t rank, uint32_t pieces) {
    return {low, (const T*)wide, scales, G, np, rank, pieces, rank % 8u == 0u && aligned(low, 16u), rank % 8u == 0u && aligned(wide, 16u)};
}

template <typename T>
NerfStatus forward(const NerfExtLinearDesc& d, const NerfExtRowGroups& r, const NerfExtAdapters& a, const void* x, const void* w, const float* bias, const void* residual, void* y, void* pre, float* mid, hipStream_t stream) {
    const Groups G{r.offsets, r.groups, d.rows};
    const bool vec = d.out_features % 8u == 0u && d.y_stride % 8u == 0u && aligned(y, 16u) && aligned(pre, 16u) && (!residual || (d.residual_stride % 8u == 0u && aligned(residual, 16u)));
    const bool y32 = d.out_dtype == NERF_EXT_F32;
    const GatheredOperands A{{w, x, d.in_features, d.x_stride, d.out_features, d.rows, d.in_features, 0u, 0u, 0u}, nullptr, r.x_rows, 0u, r.x_count};
    const RowsForwardOut<T> out{bias, (const T*)residual, y, (T*)pre, d.residual_stride, d.y_stride, d.out_features, d.rows, d.activation, y32, vec, r.y_rows, r.y_count, nullptr};
    const LowRank<T, false> more = low_rank<T, false>(mid, a.up, a.scales, G, d.out_features, a.rank, y32 && d.dtype == NERF_EXT_BF16 ? 3u : 2u);
    if (streamed(A, more, a.down, vec, r.y_rows, r.y_count, out.widest_row())) {
        NERF_HIP_TRY((launch_stream<T, false>(A, out.near(), more, StreamRanks{a.down, mid, r.y_rows, r.y_count}, stream)));
        return NERF_STATUS_OK;
    }
    NERF_HIP_TRY((launch_ranks<T, false>(G, (const T*)x, d.x_stride, r.x_rows, r.x_count, (const T*)a.down, d.in_features, a.rank, nullptr, mid, stream)));
    NERF_HIP_TRY((launch_adapter<T, false>(A, out, more, stream)));
    return NERF_STATUS_OK;
}

template <typename T>
NerfStatus backward(const NerfExtLinearDesc& d, const NerfExtRowGroups& r, const NerfExtAdapters& a, const void* x, const void* w, const void* delta, const float* mid, const void* pre, const void* add, void* dx, void* dpre, float* dmid,
                    float* ddown, float* dup, Workspace ws, hipStream_t stream) {
    const Groups G{r.offsets, r.groups, d.rows};
    const bool to_x = (dx || dpre) && d.rows;
    bool have_low   = !d.rows || !dmid;
    if (to_x) {
        const bool vec = d.in_features % 8u == 0u && (!(add || dx) || d.x_stride % 8u == 0u) && aligned(add, 16u) && aligned(dx, 16u) && aligned(pre, 16u) && aligned(dpre, 16u);
        const GatheredOperands A{{w, delta, d.in_features, d.y_stride, d.in_features, d.rows, d.out_features, 0u, 0u, 0u}, nullptr, r.y_rows, 0u, r.y_count};
        const RowsGradientOut<T> out{(const T*)add, (T*)dx, (const T*)pre, (T*)dpre, d.x_stride, d.in_features, d.rows, d.activation, vec, r.x_rows, r.x_count, nullptr};
        LowRank<T, true> more = low_rank<T, true>(dmid, a.down, nullptr, G, d.in_features, a.rank, 2u);
        if (streamed(A, more, a.up, vec, r.x_rows, r.x_count, out.widest_row())) {
            more.scales = a.scales;
            NERF_HIP_TRY((launch_stream<T, true>(A, out.near(), more, StreamRanks{a.up, dmid, r.x_rows, r.x_count}, stream)));
        } else {
            NERF_HIP_TRY((launch_ranks<T, true>(G, (const T*)delta, d.y_stride, r.y_rows, r.y_count, (const T*)a.up, d.out_features, a.rank, a.scales, dmid, stream)));
            NERF_HIP_TRY((launch_adapter<T, true>(A, out, more, stream)));
        }
        have_low = true;
    }
    if (!have_low) NERF_HIP_TRY((launch_ranks<T, true>(G, (const T*)delta, d.y_stride, r.y_rows, r.y_count, (const T*)a.up, d.out_features, a.rank, a.scales, dmid, stream)));
    if (ddown) NERF_HIP_TRY((launch_rank_sums<T>(RankSums{x, dmid, nullptr, ddown, nullptr, r.x_rows, d.x_stride, r.x_count, d.in_features, a.rank, 0u, 0u, true}, G, ws, stream)));
    if (dup) NERF_HIP_TRY((launch_rank_sums<T>(RankSums{delta, mid, a.scales, dup, nullptr, r.y_rows, d.y_stride, r.y_count, d.out_features, a.rank, 0u, 0u, false}, G, ws, stream)));
    return NERF_STATUS_OK;
}

NerfStatus check_adapters(const NerfExtAdapters* adapters, NerfExtAdapters& a, const char* fn) {
    auto refuse = [&](const char* why) {
        set_error(std::string(fn) + ": " + why);
        return NERF_STATUS_INVALID_USAGE;
    };
    if (!adapters) return refuse("null adapters");
    a = *adapters;
    if (a.rank == 0u || a.rank > (uint32_t)NERF_EXT_MAX_RANK) return refuse("rank must be 1..256");
    if (a.reserved != 0u) return refuse("reserved of the adapters must be 0");
    if (!aligned(a.down, 2u) || !aligned(a.up, 2u) || !aligned(a.scales, 4u)) return refuse("an adapter's array is not aligned to its elements");
    return NERF_STATUS_OK;
}

}  // namespace

extern "C" {

NERF_API NerfStatus nerf_ext_adapter_linear_forward(const NerfExtLinearDesc* desc, const NerfExtRowGroups* groups, const NerfExtAdapters* adapters, const void* x, const void* weight, const float* bias, const void* residual, void* y, void* pre,
                                                   float* mid, void* workspace, uint64_t workspace_bytes, void* stream) {
    NerfExtLinearDesc d;
    NerfExtRowGroups r;
    NerfExtAdapters a;
    NerfStatus s = check_desc(desc, d, "nerf_ext_adapter_linear_forward");
    if (s == NERF_STATUS_OK) s = check_groups(groups, d, r, "nerf_ext_adapter_linear_forward");
    if (s == NERF_STATUS_OK) s = check_adapters(adapters, a, "nerf_ext_adapter_linear_forward");
    if (s != NERF_STATUS_OK) return s;
    (void)workspace_bytes;
    if (d.rows == 0u) return NERF_STATUS_OK;
    NERF_CHECK_ARG(x && weight && y && mid && a.down && a.up, "nerf_ext_adapter_linear_forward: null x, weight, y, mid, down or up");
    NERF_CHECK_ARG(aligned(x, 2u) && aligned(weight, 2u) && aligned(residual, 2u) && aligned(pre, 2u) && aligned(bias, 4u) && aligned(mid, 4u) && aligned(y, d.out_dtype == NERF_EXT_F32 ? 4u : 2u),
                   "nerf_ext_adapter_linear_forward: an array is not aligned to its elements");
    NERF_CHECK_ARG(y != residual || (d.out_dtype == d.dtype && (r.y_count == 1u || d.y_stride == d.residual_stride)), "nerf_ext_adapter_linear_forward: y over residual must have its type and row stride");
    NERF_CHECK_ARG(aligned(workspace, 16u), "nerf_ext_adapter_linear_forward: workspace must be aligned to 16 bytes");
    if (d.dtype == NERF_EXT_F16) return forward<half_t>(d, r, a, x, weight, bias, residual, y, pre, mid, (hipStream_t)stream);
    return forward<bf16_t>(d, r, a, x, weight, bias, residual, y, pre, mid, (hipStream_t)stream);
}

NERF_API NerfStatus nerf_ext_adapter_linear_backward(const NerfExtLinearDesc* desc, const NerfExtRowGroups* groups, const NerfExtAdapters* adapters, const void* x, const void* weight, const void* delta, const float* mid, const void* pre,
                                                    const void* add, void* dx, void* dpre, float* dmid, float* ddown, float* dup, void* workspace, uint64_t workspace_bytes, void* stream) {
    NerfExtLinearDesc d;
    NerfExtRowGroups r;
    NerfExtAdapters a;
    NerfStatus s = check_desc(desc, d, "nerf_ext_adapter_linear_backward");
    if (s == NERF_STATUS_OK) s = check_groups(groups, d, r, "nerf_ext_adapter_linear_backward");
    if (s == NERF_STATUS_OK) s = check_adapters(adapters, a, "nerf_ext_adapter_linear_backward");
    if (s != NERF_STATUS_OK) return s;
    NERF_CHECK_ARG(dx || dpre || ddown || dup || dmid, "nerf_ext_adapter_linear_backward: no output");
    const bool low = dx || dpre || ddown;  // what dmid is needed for
    NERF_CHECK_ARG(d.rows == 0u || delta, "nerf_ext_adapter_linear_backward: null delta");
    NERF_CHECK_ARG(d.rows == 0u || dmid || !low, "nerf_ext_adapter_linear_backward: dx, dpre and ddown need dmid");
    NERF_CHECK_ARG(d.rows == 0u || a.up || !dmid, "nerf_ext_adapter_linear_backward: dmid needs up");
    NERF_CHECK_ARG(d.rows == 0u || (weight && a.down) || !(dx || dpre), "nerf_ext_adapter_linear_backward: dx and dpre need weight and down");
    NERF_CHECK_ARG(d.rows == 0u || pre || !dpre, "nerf_ext_adapter_linear_backward: dpre needs pre");
    NERF_CHECK_ARG(d.rows == 0u || x || !ddown, "nerf_ext_adapter_linear_backward: ddown needs x");
    NERF_CHECK_ARG(d.rows == 0u || mid || !dup, "nerf_ext_adapter_linear_backward: dup needs mid");
    NERF_CHECK_ARG(aligned(x, 2u) && aligned(weight, 2u) && aligned(delta, 2u) && aligned(pre, 2u) && aligned(add, 2u) && aligned(dx, 2u) && aligned(dpre, 2u) && aligned(mid, 4u) && aligned(dmid, 4u) && aligned(ddown, 4u) && aligned(dup, 4u),
                   "nerf_ext_adapter_linear_backward: an array is not aligned to its elements");
    NERF_CHECK_ARG(aligned(workspace, 16u), "nerf_ext_adapter_linear_backward: workspace must be aligned to 16 bytes");
    if (d.rows == 0u && !ddown && !dup) return NERF_STATUS_OK;
    const Workspace ws{(float*)workspace, workspace ? workspace_bytes : 0u};
    if (d.dtype == NERF_EXT_F16) return backward<half_t>(d, r, a, x, weight, delta, mid, pre, add, dx, dpre, dmid, ddown, dup, ws, (hipStream_t)stream);
    return backward<bf16_t>(d, r, a, x, weight, delta, mid, pre, add, dx, dpre, dmid, ddown, dup, ws, (hipStream_t)stream);
}

}  // extern "C"
