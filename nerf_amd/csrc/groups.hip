// groups.hip — rows put in groups by an id (include/nerf_ext.h,
// nerf_ext_group_rows): a stable counting sort.
//
//   offsets[g] = number of rows with id < g,
//   order[offsets[g] + j] = the j-th row with id g,   place[order[i]] = i,
//   rows in no group (id >= groups) behind all others.
//
// One pass counts every chunk's rows by id, one adds the counts up (over the
// chunks, then over the groups), and one finds every row's place: the counts of
// ids before its own, of its own in the chunks before, in the waves before and
// in the lanes before.  No atomic's order decides a place.  Up to 8192 rows one
// workgroup does all of it in one launch.
#include "common.hpp"

using namespace nerf_hip;

namespace {

constexpr uint32_t kThreads = 1024u, kWaves = kThreads / 64u;
constexpr uint32_t kEach = 4u, kTurn = kThreads * kEach;  // rows a turn; where one workgroup does all, twice as many
// One workgroup / three launches, us: 4096 rows in 64 groups 8.4 / 11.5, 8192 10.9 /
// 11.9, 16384 18.8 / 12.2; in 4000 groups 16 / 20, 18 / 20, 33 / 20.
constexpr uint32_t kOneRows = 8192u;

// Counters of a workgroup: where the next row of an id goes, and how many of a
// turn's rows the waves before have (two 16-bit counters a word; the last line
// has all waves').  Sized for the most groups: smaller ones for fewer groups made no
// difference (1048576 rows in 64 groups 16.0 us, in 512 19.7).
constexpr uint32_t kBins = NERF_EXT_MAX_GROUPS + 1u, kWords = (kBins + 1u) / 2u;
struct Counters {
    uint32_t start[kBins];
    uint32_t turn[kWaves + 1u][kWords];
};

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d *= 2u) {
        const uint32_t u = (uint32_t)__shfl_up((int)v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// The sums before each of `bins` values, which value(b) gives and put(b, sum)
// takes; by all threads of a workgroup, several consecutive values each.
template <uint32_t kBlock, typename Value, typename Put>
__device__ __forceinline__ void sums_before(uint32_t bins, uint32_t* lds_waves, Value value, Put put) {
    const uint32_t each = (bins + kBlock - 1u) / kBlock, first = threadIdx.x * each, wave = threadIdx.x >> 6;
    uint32_t sum = 0u;
    for (uint32_t b = first; b < min(bins, first + each); ++b) sum += value(b);
    const uint32_t to_here = wave_inclusive(sum);
    if ((threadIdx.x & 63u) == 63u) lds_waves[wave] = to_here;
    __syncthreads();
    uint32_t before = to_here - sum;
    for (uint32_t w = 0; w < wave; ++w) before += lds_waves[w];
    for (uint32_t b = first; b < min(bins, first + each); ++b) {
        const uint32_t v = value(b);
        put(b, before);
        before += v;
    }
}

// Rows [row0, row_end): their ids, counted into `counts` (LDS, cleared here).
template <uint32_t kEach>
__device__ __forceinline__ void count_rows(const uint32_t* __restrict__ ids, uint32_t row0, uint32_t row_end, uint32_t groups, uint32_t* counts) {
    for (uint32_t b = threadIdx.x; b <= groups; b += kThreads) counts[b] = 0u;
    __syncthreads();
    for (uint64_t base = row0; base < row_end; base += kThreads * kEach) {
        uint32_t id[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint64_t row = base + i * kThreads + threadIdx.x;
            id[i]              = row < row_end ? min(ids[row], groups) : ~0u;
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if (id[i] != ~0u) atomicAdd(&counts[id[i]], 1u);
    }
    __syncthreads();
}

// Places of rows [row0, row_end), S.start holding the chunk's first of every id.
template <uint32_t kEach>
__device__ __forceinline__ void place_rows(const uint32_t* __restrict__ ids, uint32_t row0, uint32_t row_end, uint32_t groups, uint32_t* __restrict__ order, uint32_t* __restrict__ place, Counters& S) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, words = (groups + 2u) / 2u;
    const uint32_t bits = 32u - (uint32_t)__builtin_clz(groups);  // of ids 0 .. groups
    constexpr uint32_t kTurn = kThreads * kEach;
    for (uint64_t base = row0; base < row_end; base += kTurn) {
        // A wave has consecutive rows, so that waves and turns are in the rows' order.
        uint32_t id[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint64_t row = base + (wave * kEach + i) * 64u + lane;
            id[i]              = row < row_end ? min(ids[row], groups) : ~0u;
        }
        for (uint32_t w = threadIdx.x; w < kWaves * words; w += kThreads) S.turn[w / words][w % words] = 0u;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if (id[i] != ~0u) atomicAdd(&S.turn[wave][id[i] / 2u], 1u << 16u * (id[i] & 1u));
        __syncthreads();
        for (uint32_t w = threadIdx.x; w < words; w += kThreads) {
            uint32_t sum = 0u;  // no carry: a turn has kTurn rows
#pragma unroll
            for (uint32_t v = 0; v < kWaves; ++v) {
                const uint32_t c = S.turn[v][w];
                S.turn[v][w]     = sum;
                sum += c;
            }
            S.turn[kWaves][w] = sum;
        }
        __syncthreads();
        volatile uint32_t* mine = S.turn[wave];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            // Lanes with the same id; those without a row are no one's.
            uint64_t same = __ballot(id[i] != ~0u);
            for (uint32_t b = 0; b < bits; ++b) {
                const uint64_t set = __ballot(id[i] >> b & 1u);
                same &= id[i] >> b & 1u ? set : ~set;
            }
            if (id[i] != ~0u) {
                const uint32_t shift = 16u * (id[i] & 1u), before = mine[id[i] / 2u] >> shift & 0xFFFFu;
                const uint32_t rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0u)), all = (uint32_t)__popcll(same);
                const uint32_t at = S.start[id[i]] + before + rank, row = (uint32_t)base + (wave * kEach + i) * 64u + lane;
                order[at] = row;
                if (place) place[row] = at;
                if (rank == 0u) atomicAdd(&S.turn[wave][id[i] / 2u], all << shift);
            }
            // The wave's next rows read what its leaders have added.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        for (uint32_t b = threadIdx.x; b <= groups; b += kThreads) S.start[b] += S.turn[kWaves][b / 2u] >> 16u * (b & 1u) & 0xFFFFu;
        __syncthreads();
    }
}

__global__ __launch_bounds__(kThreads) void k_group_one(const uint32_t* __restrict__ ids, uint32_t rows, uint32_t groups, uint32_t* __restrict__ offsets, uint32_t* __restrict__ order, uint32_t* __restrict__ place) {
    __shared__ Counters S;
    __shared__ uint32_t waves[kWaves];
    uint32_t* counts = &S.turn[0][0];
    static_assert((kWaves + 1u) * kWords >= kBins);
    count_rows<2u * kEach>(ids, 0u, rows, groups, counts);
    sums_before<kThreads>(groups + 1u, waves, [&](uint32_t b) { return counts[b]; }, [&](uint32_t b, uint32_t sum) {
        S.start[b] = sum;
        offsets[b] = sum;
    });
    __syncthreads();
    place_rows<2u * kEach>(ids, 0u, rows, groups, order, place, S);
}

// What the passes of more rows leave for each other.
struct Passes {
    uint32_t* totals;  // [groups + 1]
    uint32_t* counts;  // [chunks][groups + 1], then the counts of the chunks before
    uint32_t rows, groups, chunks, chunk;
};

__global__ __launch_bounds__(kThreads) void k_group_count(const uint32_t* __restrict__ ids, Passes P) {
    __shared__ uint32_t counts[kBins];
    const uint32_t row0 = blockIdx.x * P.chunk;
    count_rows<kEach>(ids, row0, min(P.rows, row0 + P.chunk), P.groups, counts);
    for (uint32_t b = threadIdx.x; b <= P.groups; b += kThreads) P.counts[(uint64_t)blockIdx.x * (P.groups + 1u) + b] = counts[b];
}

// 32 ids a workgroup, the chunks in 32 slices.
constexpr uint32_t kSlices = 32u, kIds = 32u;
__global__ __launch_bounds__(kIds * kSlices) void k_group_scan(Passes P) {
    __shared__ uint32_t slice_sum[kSlices][kIds];
    const uint32_t bins = P.groups + 1u, b = blockIdx.x * kIds + threadIdx.x % kIds, slice = threadIdx.x / kIds;
    const uint32_t each = (P.chunks + kSlices - 1u) / kSlices, first = slice * each, end = min(P.chunks, first + each);
    uint32_t sum = 0u;
    if (b < bins) {
#pragma unroll 8
        for (uint32_t c = first; c < end; ++c) sum += P.counts[(uint64_t)c * bins + b];
    }
    slice_sum[slice][threadIdx.x % kIds] = sum;
    __syncthreads();
    uint32_t before = 0u;
    for (uint32_t s = 0; s < slice; ++s) before += slice_sum[s][threadIdx.x % kIds];
    if (b >= bins) return;
#pragma unroll 8
    for (uint32_t c = first; c < end; ++c) {
        const uint32_t v = P.counts[(uint64_t)c * bins + b];
        P.counts[(uint64_t)c * bins + b] = before;
        before += v;
    }
    if (slice == kSlices - 1u) P.totals[b] = before;
}

// Every workgroup adds the totals up for itself (a launch of its own, or a wait for
// the last workgroup of the pass before, takes longer: 1048576 rows, 4096 groups
// 68 us with the latter).
__global__ __launch_bounds__(kThreads) void k_group_place(const uint32_t* __restrict__ ids, Passes P, uint32_t* __restrict__ offsets, uint32_t* __restrict__ order, uint32_t* __restrict__ place) {
    __shared__ Counters S;
    __shared__ uint32_t waves[kWaves];
    const uint32_t row0 = blockIdx.x * P.chunk;
    uint32_t* totals    = &S.turn[0][0];
    for (uint32_t b = threadIdx.x; b <= P.groups; b += kThreads) {
        totals[b]  = P.totals[b];
        S.start[b] = P.counts[(uint64_t)blockIdx.x * (P.groups + 1u) + b];
    }
    __syncthreads();
    sums_before<kThreads>(P.groups + 1u, waves, [&](uint32_t b) { return totals[b]; }, [&](uint32_t b, uint32_t sum) {
        S.start[b] += sum;
        if (blockIdx.x == 0u) offsets[b] = sum;
    });
    __syncthreads();
    place_rows<kEach>(ids, row0, min(P.rows, row0 + P.chunk), P.groups, order, place, S);
}

NerfStatus group_rows(const uint32_t* ids, uint32_t rows, uint32_t groups, uint32_t* offsets, uint32_t* order, uint32_t* place, uint32_t* workspace, uint64_t words, hipStream_t stream) {
    // Chunks: two a CU at most, as many as the workspace holds.
    const uint64_t bins = groups + 1u, held = words > bins ? (words - bins) / bins : 0u;
    const uint64_t chunks = std::min<uint64_t>({held, 2u * device_cu_count(), (rows + kTurn - 1u) / kTurn});
    if (rows <= kOneRows || chunks <= 1u) {
        k_group_one<<<1, kThreads, 0, stream>>>(ids, rows, groups, offsets, order, place);
        NERF_LAUNCH_CHECK("k_group_one");
        return NERF_STATUS_OK;
    }
    const uint32_t chunk = (uint32_t)((rows + chunks * kTurn - 1u) / (chunks * kTurn)) * kTurn;
    const Passes P{workspace, workspace + bins, rows, groups, (rows + chunk - 1u) / chunk, chunk};
    k_group_count<<<P.chunks, kThreads, 0, stream>>>(ids, P);
    NERF_LAUNCH_CHECK("k_group_count");
    k_group_scan<<<groups / kIds + 1u, kIds * kSlices, 0, stream>>>(P);
    NERF_LAUNCH_CHECK("k_group_scan");
    k_group_place<<<P.chunks, kThreads, 0, stream>>>(ids, P, offsets, order, place);
    NERF_LAUNCH_CHECK("k_group_place");
    return NERF_STATUS_OK;
}

}  // namespace

extern "C" {

NERF_API NerfStatus nerf_ext_group_rows(const uint32_t* ids, uint32_t rows, uint32_t groups, uint32_t* offsets, uint32_t* order, uint32_t* place, void* workspace, uint64_t workspace_bytes, void* stream) {
    NERF_CHECK_ARG(groups >= 1u && groups <= (uint32_t)NERF_EXT_MAX_GROUPS, "nerf_ext_group_rows: groups must be 1..4096");
    NERF_CHECK_ARG(rows <= 1u << 30, "nerf_ext_group_rows: more than 2^30 rows");
    NERF_CHECK_ARG(offsets && (rows == 0u || (ids && order)), "nerf_ext_group_rows: null ids, offsets or order");
    auto aligned = [](const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1u)) == 0u; };
    NERF_CHECK_ARG(aligned(ids, 4u) && aligned(offsets, 4u) && aligned(order, 4u) && aligned(place, 4u), "nerf_ext_group_rows: an array is not aligned to its elements");
    NERF_CHECK_ARG(aligned(workspace, 16u), "nerf_ext_group_rows: workspace must be aligned to 16 bytes");
    const uint64_t words = workspace ? workspace_bytes / 4u : 0u;
    return group_rows(ids, rows, groups, offsets, order, place, (uint32_t*)workspace, words, (hipStream_t)stream);
}

}  // extern "C"
