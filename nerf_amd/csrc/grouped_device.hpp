// grouped_device.hpp — rows in groups, as the layers with weights of their own
// for every group (grouped.hip) and those with adapters (adapter.hip) have them:
// which group a tile belongs to, outputs whose rows an index names, and the join
// of sums over a group's rows that were split.
//
// Positions 0 .. rows - 1 are in the groups' order: group g has those from
// offsets[g] to offsets[g + 1].  The offsets are in device memory, so neither
// the host nor the launch knows how many tiles a group has.  With tiles of B
// positions, group g gets the tile numbers from offsets[g] / B + g (rounded
// down) on: at least as many as it needs, since
//   ceil((b - a) / B) <= floor(b / B) - floor(a / B) + 1,
// and rows / B + groups in all, at most one a group of them empty.  A workgroup
// finds its group by one search and no table is made.
// Offsets are clamped to rows and rows of an index compared with the array's, so
// no content of theirs leads out of the arrays.
#pragma once

#include "linear_device.hpp"
#include "offsets.hpp"

namespace nerf_hip {
namespace grouped {

using namespace linear;

struct Groups {
    const uint32_t* offsets;
    uint32_t count, rows;
    __device__ __forceinline__ uint32_t offset(uint32_t g) const { return min(offsets[g], rows); }
};

// How many of n ascending keys are at most `s`, found by the wave together.
template <typename Key>
__device__ __forceinline__ uint32_t count_at_most(uint32_t n, uint32_t s, Key key) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t first = 0u;
    while (n > 64u) {
        const uint32_t step = (n + 63u) / 64u, at = lane * step;
        const uint32_t c = (uint32_t)__popcll(__ballot(at < n && key(first + at) <= s));
        if (c == 0u) return first;
        first += (c - 1u) * step + 1u;
        n = min(step - 1u, n - (c - 1u) * step - 1u);
    }
    return first + (uint32_t)__popcll(__ballot(lane < n && key(first + lane) <= s));
}

// Positions [q0, end) of group g; q0 >= end: nothing to do.
struct Part {
    uint32_t group, q0, end, number;  // number: of the part within its group
};

// Part number `s` of the parts of `size` positions each.  Every group has a first part
// (number 0), also one without positions; numbers before the first group's, where
// offsets[0] > 0, are of no group's first part.
__device__ __forceinline__ Part part_of(const Groups& G, uint32_t size, uint32_t s) {
    const uint32_t c = count_at_most(G.count, s, [&](uint32_t g) { return G.offset(g) / size + g; });
    if (c == 0u) return {0u, 0u, 0u, 1u};
    const uint32_t g = __builtin_amdgcn_readfirstlane(c - 1u), begin = G.offset(g), end = G.offset(g + 1u), number = s - (begin / size + g);
    const uint64_t q0 = begin + (uint64_t)number * size;
    return {g, q0 < end ? (uint32_t)q0 : end, end, number};
}
__device__ __forceinline__ uint32_t part_count(const Groups& G, uint32_t size) { return G.offset(G.count) / size + G.count; }
// The same for fewer rows than groups, by position: every size-th of a group has a
// part.
__device__ __forceinline__ Part part_at(const Groups& G, uint32_t size, uint32_t position) {
    const uint32_t c = count_at_most(G.count, position, [&](uint32_t g) { return G.offset(g); });
    if (c == 0u) return {0u, 0u, 0u, 0u};
    const uint32_t g = __builtin_amdgcn_readfirstlane(c - 1u), begin = G.offset(g), end = G.offset(g + 1u);
    const bool first = position >= begin && position < end && (position - begin) % size == 0u;
    return {g, first ? position : end, end, 0u};
}
// Which of the two, and how many parts there may be.
struct Parts {
    uint32_t most;
    bool by_position;
};
inline Parts parts_of(uint32_t rows, uint32_t groups, uint32_t size) {
    const uint32_t most = rows / size + groups;
    return rows < most ? Parts{rows, true} : Parts{most, false};
}

// A grid has fewer than 2^32 threads in x: workgroups beyond 2^20 go on in y.
inline dim3 grid_of(uint64_t blocks) { return blocks <= 1u << 20 ? dim3((uint32_t)blocks) : dim3(1u << 20, (uint32_t)((blocks + (1u << 20) - 1u) >> 20)); }
__device__ __forceinline__ uint32_t block_number() { return blockIdx.y * gridDim.x + blockIdx.x; }

// Tile of a workgroup: p the faster, in bands of four parts (see k_product in
// linear.hip), a chip's workgroups in a row.
struct GroupTile {
    uint32_t tile_p;
    Part part;
};
__device__ __forceinline__ GroupTile group_tile(const Groups& G, uint32_t size, uint32_t tiles_p, bool by_position, uint32_t most) {
    const uint32_t parts = by_position ? most : min(most, part_count(G, size));
    const uint32_t block = block_number();
    if (block >= parts * tiles_p) return {0u, {0u, 0u, 0u, 0u}};
    const uint32_t t = chip_tile(block, parts * tiles_p), band = tiles_p > 4u ? 4u : 1u;
    const uint32_t first = t / (band * tiles_p) * band, high = min(band, parts - first), in_band = t - first * tiles_p;
    const uint32_t s = first + in_band % high;
    return {in_band / high, by_position ? part_at(G, size, s) : part_of(G, size, s)};
}

// ----------------------------------------------------------------- outputs
// Eight values from p of a row, `n` of them inside; what Rows does, for rows
// anywhere in an array of any size.
template <typename E>
__device__ __forceinline__ uintx4 load_eight(const E* row, uint32_t p, uint32_t n, bool vec, bool rows_of_eight) {
    static_assert(sizeof(E) == 2);
    uintx4 o;
    if (vec) {
        o = *reinterpret_cast<const uintx4*>(row + (n ? p : 0u));
    } else if (rows_of_eight) {
        __builtin_memcpy(&o, row + (n ? p + n - 8u : 0u), 16);
    } else {
        const short* s = reinterpret_cast<const short*>(row);
        short8_t v;
#pragma unroll
        for (uint32_t r = 0; r < 8u; ++r) v[r] = s[r < n ? p + r : 0u];
        o = __builtin_bit_cast(uintx4, v);
    }
    return o;
}
template <typename E>
__device__ __forceinline__ void store_eight(E* row, uint32_t p, uint32_t n, bool vec, const floatx8& v) {
    E* at = row + p;
    if constexpr (sizeof(E) == 4) {
        const floatx4 lo = v.lo, hi = v.hi;
        if (vec && n) {
            reinterpret_cast<floatx4*>(at)[0] = lo;
            reinterpret_cast<floatx4*>(at)[1] = hi;
        } else if (n == 8u) {
            __builtin_memcpy(at, &lo, 16);
            __builtin_memcpy(at + 4, &hi, 16);
        } else {
#pragma unroll
            for (uint32_t r = 0; r < 8u; ++r)
                if (r < n) at[r] = v[r];
        }
    } else {
        const typename Vec<E>::x8 h = __builtin_convertvector(v, typename Vec<E>::x8);
        if (vec && n) {
            *reinterpret_cast<typename Vec<E>::x8*>(at) = h;
        } else if (n == 8u) {
            __builtin_memcpy(at, &h, 16);
        } else {
#pragma unroll
            for (uint32_t r = 0; r < 8u; ++r)
                if (r < n) at[r] = h[r];
        }
    }
}

// The epilogues get rows of a tile and look their place in the arrays up in LDS
// (kNoRow: nothing is written).  Threads without outputs (n = 0) may name rows
// beyond the tile, which have no place.  of_group(): what belongs to the tile's group.
template <typename T>
struct RowsForwardOut {
    const float* bias;
    const T* residual;
    void* y;
    T* pre;
    uint64_t ldr, ldy;
    uint32_t np, nq, act;
    bool y32, vec;
    const uint32_t* index;
    uint32_t count;
    const uint32_t* rows;
    struct Aux {
        uintx4 residual;
    };
    static constexpr bool kBias = true;

    // The same for rows within 32-bit offsets, and how many 16-bit values a row has.
    ForwardOut<T> near() const { return {bias, residual, y, pre, ldr, ldy, np, nq, act, y32, vec}; }
    uint64_t widest_row() const { return std::max({(y32 ? 2u : 1u) * ldy, residual ? ldr : 0u, (uint64_t)np}); }
    __device__ __forceinline__ void of_group(uint32_t g) {
        if (bias) bias += (uint64_t)g * np;
    }
    __device__ __forceinline__ Aux load(uint32_t, uint32_t row, uint32_t p, uint32_t n) const {
        if (!residual) return {uintx4{0u, 0u, 0u, 0u}};
        const uint32_t r = n ? rows[row] : kNoRow;
        return {load_eight<T>(residual + (r != kNoRow ? r : 0u) * ldr, p, r != kNoRow ? n : 0u, vec, np >= 8u)};
    }
    __device__ __forceinline__ void put(uint32_t, uint32_t row, uint32_t p, uint32_t n, floatx8 z, const floatx8& b, const Aux& a) const {
        const uint32_t r = n ? rows[row] : kNoRow;
        if (r == kNoRow) return;
        z += b;
        if (pre) store_eight<T>(pre + (uint64_t)r * np, p, n, vec, z);
        act_values(act, z);
        if (residual) z += widen<T>(a.residual, n, vec, np >= 8u);
        if (y32) store_eight<float>((float*)y + r * ldy, p, n, vec, z);
        else store_eight<T>((T*)y + r * ldy, p, n, vec, z);
    }
};

template <typename T>
struct RowsGradientOut {
    const T* add;
    T* dx;
    const T* pre;
    T* dpre;
    uint64_t ldx;
    uint32_t np, nq, act;
    bool vec;
    const uint32_t* index;
    uint32_t count;
    const uint32_t* rows;
    struct Aux {
        uintx4 add, pre;
    };
    static constexpr bool kBias = false;

    InputGradientOut<T> near() const { return {add, dx, pre, dpre, ldx, np, nq, act, vec}; }
    uint64_t widest_row() const { return std::max(ldx, (uint64_t)np); }
    __device__ __forceinline__ void of_group(uint32_t) {}
    __device__ __forceinline__ Aux load(uint32_t, uint32_t row, uint32_t p, uint32_t n) const {
        Aux a{};
        const uint32_t r = n ? rows[row] : kNoRow, at = r != kNoRow ? r : 0u;
        if (r == kNoRow) n = 0u;
        if (add) a.add = load_eight<T>(add + at * ldx, p, n, vec, np >= 8u);
        if (dpre) a.pre = load_eight<T>(pre + (uint64_t)at * np, p, n, vec, np >= 8u);
        return a;
    }
    __device__ __forceinline__ void put(uint32_t, uint32_t row, uint32_t p, uint32_t n, floatx8 g, const floatx8&, const Aux& a) const {
        const uint32_t r = n ? rows[row] : kNoRow;
        if (r == kNoRow) return;
        if (add) g += widen<T>(a.add, n, vec, np >= 8u);
        if (dx) store_eight<T>(dx + r * ldx, p, n, vec, g);
        if (dpre) {
            floatx8 s = widen<T>(a.pre, n, vec, np >= 8u);
            act_slopes(act, s);
            store_eight<T>(dpre + (uint64_t)r * np, p, n, vec, g * s);
        }
    }
};

// Sums by position in 32 bits, times the group's scale.
struct PositionOut {
    float* out;  // dense [rows][np]
    const float* scales;
    uint32_t np, nq;
    bool vec;
    float scale;
    struct Aux {};
    static constexpr bool kBias = false;
    __device__ __forceinline__ void of_group(uint32_t g) { scale = scales ? scales[g] : 1.0f; }
    __device__ __forceinline__ Aux load(uint32_t, uint32_t, uint32_t, uint32_t) const { return {}; }
    __device__ __forceinline__ void put(uint32_t q0, uint32_t row, uint32_t p, uint32_t n, const floatx8& v, const floatx8&, const Aux&) const { Rows<float>(out, q0, np).store(row, p, n, vec, v * scale); }
};

template <typename Out>
constexpr bool kHasRows = !std::is_same_v<Out, PositionOut>;
// The rows of a tile's outputs into LDS; the caller's next barrier is theirs.
template <uint32_t kBQ, typename Out>
__device__ __forceinline__ void find_rows(Out& out, uint32_t* lds, uint32_t q0, uint32_t end) {
    if constexpr (kHasRows<Out>) {
        if (threadIdx.x < kBQ) lds[threadIdx.x] = gathered_row(out.index, out.count, q0 + threadIdx.x, end);
        out.rows = lds;
    }
}

// -------------------------------------------------------------------- sums
// Parts are of uneven length, so their tiles are dealt to the eight chips in turn, a
// few at a time that share operands: a whole part's (32 at most) where there are
// many parts, else an eighth, so that no chip has the longest group to itself.
// (16384 x 2048 -> 4096 in 8 groups of up to 6200 rows, sums alone: 770 us with a
// chip's tiles in a row, 320 dealt by eighths; 262144 x 256 -> 256 in 64 groups
// 97 us by single tiles, 87 by parts.)  A workgroup beyond the last tile gets a
// number beyond it.
inline __host__ __device__ uint32_t dealt_at_once(uint32_t parts, uint32_t tiles) {
    const uint32_t u = parts >= 64u ? tiles : tiles / 8u;
    return u < 1u ? 1u : u > 32u ? 32u : u;
}
__device__ __forceinline__ uint32_t dealt_tile(uint32_t b, uint32_t parts, uint32_t tiles) {
    const uint32_t u = dealt_at_once(parts, tiles), j = b / 8u;
    return (j / u * 8u + b % 8u) * u + j % u;
}
inline uint64_t dealt_blocks(uint32_t parts, uint32_t tiles) {
    const uint64_t turn = 8u * dealt_at_once(parts, tiles);
    return ((uint64_t)parts * tiles + turn - 1u) / turn * turn;
}

// Sums over a group's rows are made of parts of `size` positions: the first part
// is in the output, part t > 0 of group g in place offsets[g] / size + t - 1 of
// the others (no two parts share one, and there are rows / size of them at most,
// by the inequality above).
__device__ __forceinline__ uint64_t place_of(const Groups& G, const Part& part, uint32_t size) { return (uint64_t)(G.offset(part.group) / size) + part.number - 1u; }

// ------------------------------------------------------------------- host
constexpr uint32_t kMaxGroups = NERF_EXT_MAX_GROUPS;

// What NerfExtRowGroups says, with its defaults filled in.
NerfStatus check_groups(const NerfExtRowGroups* groups, const NerfExtLinearDesc& d, NerfExtRowGroups& out, const char* fn);

// out[g * length + e] (and sums[g * sums_length + e]) += their parts.
hipError_t launch_join(const Groups& G, uint32_t size, float* out, const float* parts, uint64_t length, float* sums, const float* sum_parts, uint32_t sums_length, hipStream_t stream);

// Positions a part of a sum over rows: as many parts as give `fill` workgroups with
// `tiles` of them a part, 256 positions at least, as few as the workspace holds.
inline uint32_t part_size(uint32_t rows, uint64_t tiles, uint64_t fill, uint64_t bytes_a_part, uint64_t workspace_bytes) {
    const uint64_t wanted = std::max<uint64_t>(1u, fill / std::max<uint64_t>(1u, tiles)), held = workspace_bytes / bytes_a_part;
    uint64_t size = std::max<uint64_t>(256u, (rows + wanted - 1u) / wanted);
    if (rows / size > held) size = rows / (held + 1u) + 1u;  // rows / size <= held
    return (uint32_t)std::min<uint64_t>((size + kBK - 1u) / kBK * kBK, 1u << 31);
}

// mid[i] = scale x_i A_g^T by position in 32 bits (kPT: d_i B_g): what grouped.hip
// has for the adapters.
template <typename T, bool kPT>
hipError_t launch_ranks(const Groups& G, const T* x, uint64_t ldx, const uint32_t* index, uint32_t count, const T* weight, uint32_t features, uint32_t rank, const float* scales, float* out, hipStream_t stream);

}  // namespace grouped
}  // namespace nerf_hip
