// grouped.hip — linear layers with weights of their own for every group of rows
// (include/nerf_ext.h, nerf_ext_grouped_linear_*): the products of linear.hip,
// each tile of rows with its group's weights.
//
//   forward:   z_i = W_g x_i + b_g,  y_i = act(z_i) + r_i         i in group g
//   backward:  g_i = d_i W_g + a_i,  dx = g,  dpre = g act'(pre),
//              dW_g = sum_i d_i x_i^T,  db_g = sum_i d_i
//
// A tile is of one group (grouped_device.hpp says which), so the work is that of
// the rows rounded up to tiles, group by group.
#include "grouped_device.hpp"

using namespace nerf_hip;
using namespace nerf_hip::grouped;

namespace {

// Output tiles of kBP x kBQ, see product().  A tile's rows are looked up once, into
// LDS; rows of an operand are asked for a tile of k ahead, since each is two loads
// that wait for each other.  With 256 -> 256 fp16, residual and pre, 262144 rows in 64
// groups, memory bounds it: 130 us, 4.1 TB/s (weights of a group are in L2 for its
// rows, so a kernel that streams the rows past them in registers was 3 % faster
// here and slower with many groups; it is not built).  With 4096 -> 4096 bf16 the
// matrix instructions do: 16384 rows in 8 groups 550-565 us, 1.0 PFLOP/s, of which a
// sixth is the last round of tiles, not full, and tiles half beyond a group's end.
template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, uint32_t kDepth, bool kPT, Mode kMode, bool kGather, typename Out>
__global__ __launch_bounds__(kWP * kWQ * 64u) void k_grouped(GatheredOperands A, Out out, Groups G, Parts parts) {
    __shared__ uint32_t rows[kHasRows<Out> ? kBQ : 1u];
    const GroupTile tile = group_tile(G, kBQ, A.tiles_p, parts.by_position, parts.most);
    const Part& part = tile.part;
    if (part.q0 >= part.end) return;
    find_rows<kBQ>(out, rows, part.q0, part.end);
    out.of_group(part.group);
    out.nq = A.nq = part.end;
    product<T, kBP, kBQ, kWP, kWQ, kDepth, kPT, false, kMode, kGather>(A, out, Place{tile.tile_p * kBP, part.q0, 0u, A.nk, kPT ? 0u : part.group * A.np, kPT ? part.group * A.nk : 0u});
}

// The same with few tiles, each one's k over a workgroup's waves, which bounds a call
// by one pass of loads (8 rows in as many of 64 groups, 256 -> 256: 4.2-5.0 us, the
// launch being 4).  kWhole: whole steps and rows that start at even values.
template <typename T, uint32_t kF, bool kPT, bool kWhole, typename Out>
__global__ __launch_bounds__(kFewWaves * 64u) void k_grouped_few(GatheredOperands A, Out out, Groups G, Parts parts) {
    __shared__ floatx4 lds[few_lds(kF, kF) / 16u];
    __shared__ uint32_t rows[kHasRows<Out> ? 16u * kF : 1u];
    const GroupTile tile = group_tile(G, 16u * kF, A.tiles_p, parts.by_position, parts.most);
    const Part& part = tile.part;
    if (part.q0 >= part.end) return;
    out.of_group(part.group);
    out.nq = A.nq = part.end;
    few_tile<T, kF, kF, kPT, false, !kWhole, true, kWhole>(A, out, Place{tile.tile_p * 16u * kF, part.q0, 0u, A.nk, kPT ? 0u : part.group * A.np, kPT ? part.group * A.nk : 0u}, reinterpret_cast<char*>(lds), nullptr, rows);
}

// Weights or rows of fewer than eight values in all: a thread computes eight
// outputs of a position from memory.
template <typename T, bool kPT, typename Out>
__global__ __launch_bounds__(64) void k_grouped_tiny(GatheredOperands A, Out out, Groups G) {
    __shared__ uint32_t rows[1];
    for (uint32_t position = blockIdx.x; position < G.rows; position += gridDim.x) {
        const Part part = part_at(G, 1u, position);
        if (part.q0 >= part.end) continue;
        Out mine = out;
        __syncthreads();
        find_rows<1u>(mine, rows, position, position + 1u);
        __syncthreads();
        mine.of_group(part.group);
        const uint32_t from = gathered_row(A.q_index, A.q_count, position, position + 1u);
        for (uint32_t p = 8u * threadIdx.x; p < A.np; p += 512u) {
            const uint32_t n = min(8u, A.np - p);
            const typename Out::Aux aux = mine.load(position, 0u, p, n);
            floatx8 v = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, b = v;
            for (uint32_t k = 0; k < A.nk; ++k) {
                const float x = from == kNoRow ? 0.0f : (float)((const T*)A.q)[from * A.ldq + k];
#pragma unroll
                for (uint32_t r = 0; r < 8u; ++r)
                    if (r < n) v[r] += x * (float)((const T*)A.p)[kPT ? ((uint64_t)part.group * A.nk + k) * A.ldp + p + r : ((uint64_t)part.group * A.np + p + r) * A.ldp + k];
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

// dW_g, and db_g with it: sums over parts of `size` rows of a group, both operands by
// the transposing read.  Every product is of two rows' values that are read again
// for each tile across, so it is bound by memory where a layer is narrow (262144
// rows in 64 groups, 256 x 256: 88 us, 3.1 TB/s, and 9 for the join) and by the matrix
// instructions where it is wide (16384 rows in 8 groups, 2048 x 4096: 326 us, 0.84
// PFLOP/s: the groups' uneven rows leave CUs without work at the end).
template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, Mode kMode, bool kGather>
__global__ __launch_bounds__(kWP * kWQ * 64u) void k_grouped_sums(GatheredOperands A, SumOut out, Groups G, uint32_t size, uint32_t most, float* sum_parts) {
    const uint32_t tiles = A.tiles_p * A.tiles_q, t = dealt_tile(block_number(), most, tiles);
    if (t >= most * tiles) return;
    const Part part = part_of(G, size, t / tiles);
    if (part.q0 >= part.end && part.number) return;
    const uint64_t length = (uint64_t)A.np * A.nq;
    if (part.number) {
        const uint64_t at = place_of(G, part, size);
        out.out = out.parts + at * length;
        if (out.row_sums) out.row_sums = sum_parts + at * A.nq;
    } else {
        out.out += part.group * length;
        if (out.row_sums) out.row_sums += (uint64_t)part.group * A.nq;
    }
    product<T, kBP, kBQ, kWP, kWQ, 2u, true, true, kMode, kGather>(A, out, Place{t % tiles % A.tiles_p * kBP, t % tiles / A.tiles_p * kBQ, part.q0, min(part.end, part.q0 + size), 0u, 0u});
}

// Sums of operands of fewer than eight values in all: one thread an output.
template <typename T>
__global__ __launch_bounds__(256) void k_grouped_tiny_sums(GatheredOperands A, SumOut out, Groups G) {
    const uint64_t at = block_number() * 256ull + threadIdx.x, total = (uint64_t)G.count * A.np * A.nq;
    if (at >= total) return;
    const uint32_t p = (uint32_t)(at % A.np), q = (uint32_t)(at / A.np % A.nq), g = (uint32_t)(at / A.np / A.nq);
    float v = 0.0f, s = 0.0f;
    for (uint32_t i = G.offset(g), end = G.offset(g + 1u); i < end; ++i) {
        const uint32_t a = gathered_row(A.p_index, A.p_count, i, end), b = gathered_row(A.q_index, A.q_count, i, end);
        const float x = a == kNoRow ? 0.0f : (float)((const T*)A.p)[a * A.ldp + p], d = b == kNoRow ? 0.0f : (float)((const T*)A.q)[b * A.ldq + q];
        v += x * d;
        s += d;
    }
    out.out[at] = v;
    if (out.row_sums && p == 0u) out.row_sums[(uint64_t)g * A.nq + q] = s;
}

// The parts of a group added to its first, in their order.
__global__ __launch_bounds__(256) void k_grouped_join(Groups G, uint32_t size, float* out, const float* parts, uint64_t length, float* sums, const float* sum_parts, uint32_t sums_length, uint32_t blocks) {
    const uint32_t g = blockIdx.x / blocks, begin = G.offset(g), end = G.offset(g + 1u);
    if (end <= begin || end - begin <= size) return;
    const uint32_t count = (end - begin + size - 1u) / size, first = begin / size;
    for (uint64_t e = (blockIdx.x % blocks) * 256ull + threadIdx.x; e < length + sums_length; e += blocks * 256ull) {
        const bool sum = e >= length;
        const uint64_t stride = sum ? sums_length : length, at = sum ? e - length : e;
        const float* from = (sum ? sum_parts : parts) + first * stride + at;
        float* to         = (sum ? sums : out) + g * stride + at;
        float v = *to;
#pragma unroll 8
        for (uint32_t t = 0; t < count - 1u; ++t) v += from[t * stride];
        *to = v;
    }
}

// ------------------------------------------------------------------- host
template <typename T, bool kPT, typename Out>
hipError_t launch_grouped(GatheredOperands A, Out out, const Groups& G, hipStream_t stream) {
    const uint64_t weights = (uint64_t)G.count * A.np * A.nk, values = (uint64_t)(A.q_count - 1u) * A.ldq + A.nk;
    if (weights < 8u || values < 8u) {
        k_grouped_tiny<T, kPT, Out><<<std::min(G.rows, 64u * device_cu_count()), 64, 0, stream>>>(A, out, G);
        return hipGetLastError();
    }
    auto launch = [&](auto kernel, uint32_t bp, uint32_t bq, uint32_t threads) {
        const Parts parts = parts_of(G.rows, G.count, bq);
        A.tiles_p         = ceil_div(A.np, bp);
        kernel<<<grid_of((uint64_t)parts.most * A.tiles_p), threads, 0, stream>>>(A, out, G, parts);
        return hipGetLastError();
    };
    const bool gather = A.q_index != nullptr;
    const bool words  = !whole_chunks(A.p, A.ldp, kPT ? A.np : A.nk) || !whole_chunks(A.q, A.ldq, A.nk) || (gather && !near(A.q_count, A.ldq));
    const uint64_t cus = device_cu_count();
    // Tiles that the rows can make, group by group, and about how many they do.
    auto tiles   = [&](uint32_t b) { return (uint64_t)ceil_div(A.np, b) * parts_of(G.rows, G.count, b).most; };
    auto on_mean = [&](uint32_t b) { return (uint64_t)ceil_div(A.np, b) * (G.rows / b + G.count / 2u); };
    // Fewer tiles than CUs: the k of a tile over a workgroup's waves.  us, few of 16 / of
    // 32 / tiles of 64, fp16, 4096 -> 1024: 32 rows 1 group (192, 64 tiles) 11 / 18 / 18;
    // 32 rows 4 groups (384, 160) 18 / 16.5 / 18.6; 64 rows 8 groups (768, 320) 26 / 30 /
    // 19.  1024 -> 1024: 1 row 5.5 / 6.5 / 7.5; 32 rows 4 groups 7.6 / 7.1 / 7.8; 256 rows 8
    // groups 18 / 12 / 8.7.
    if (A.nk <= kFewMaxK) {
        auto few = [&](auto f) {
            const bool whole = A.nk % 32u == 0u && (!kPT || A.np % (16u * f()) == 0u) && !odd_rows(A.p, A.ldp) && !odd_rows(A.q, A.ldq) && ((uint64_t)A.np * A.nk) % 2u == 0u;
            if (whole) return launch(k_grouped_few<T, f(), kPT, true, Out>, 16u * f(), 16u * f(), kFewWaves * 64u);
            return launch(k_grouped_few<T, f(), kPT, false, Out>, 16u * f(), 16u * f(), kFewWaves * 64u);
        };
        if (tiles(16u) <= cus) return few(std::integral_constant<uint32_t, 1u>{});
        if (tiles(32u) <= cus) return few(std::integral_constant<uint32_t, 2u>{});
    }
    const uint32_t mean = G.rows / G.count;
    if constexpr (!kHasRows<Out>) {
        if (words) return launch(k_grouped<T, 64, 64, 2, 2, 2, kPT, kByWords, true, Out>, 64u, 64u, 256u);
        return gather ? launch(k_grouped<T, 64, 64, 2, 2, 4, kPT, kDirect, true, Out>, 64u, 64u, 256u) : launch(k_grouped<T, 64, 64, 2, 2, 4, kPT, kDirect, false, Out>, 64u, 64u, 256u);
    } else {
        // us, tiles of 64 / of 128, fp16 256 -> 256: 4096 rows in 64 groups 7.3 / 10.5, 8192
        // 11.9 / 12.0, in 128 13.5 / 13.7, 16384 in 64 17 / 14, 131072 in 16 108 / 69; bf16
        // 2048 -> 2048: 2048 rows in 8 groups 44 / 36, 1024 in 32 67 / 90, 2048 83 / 90,
        // 4096 123 / 100.  Where there may be so many tiles that most have no rows, fewer numbers
        // count for more than full tiles: 4096 rows in 1024 groups 35 / 34, 16384 in 4096 153 /
        // 137, 262144 in 4096 317 / 245, the same if 8 of them have all the rows 388 / 281.
        // By words a tile of 128 waits for its one buffer, and pays with many products only:
        // 255 -> 255, 65536 rows in 512 groups 81 / 97, 262144 246 / 245; 1023 -> 1023, 8192 in 16
        // 77 / 90, 16384 147 / 141, in 128 207 / 209, 65536 in 64 542 / 452, 32768 in 512 498 / 562.
        const uint64_t products = (uint64_t)G.rows * A.np * A.nk;
        const bool by_128 = A.np > 64u && tiles(128u) >= cus && (words ? mean >= 128u && products >= 1ull << 34 : mean >= 64u || tiles(128u) >= 8u * cus);
        if (words) return by_128 ? launch(k_grouped<T, 128, 128, 2, 2, 2, kPT, kByWords, true, Out>, 128u, 128u, 256u) : launch(k_grouped<T, 64, 64, 2, 2, 2, kPT, kByWords, true, Out>, 64u, 64u, 256u);
        // A CU has one tile of 256 at a time, as long as 2.75 of 128 take it, and the last
        // round of them is seldom full.  us, 128 / 256, bf16: 4096 -> 4096, 16384 rows in 8
        // groups (5 rounds for 16.5) 626 / 584, 8192 rows (3 for 8.5) 364 / 327; 2048 -> 2048,
        // 16384 rows in 16 (3 for 8.5) 197 / 194, 8192 rows in 8 (2 for 4.25) 97 / 126, in 64
        // groups 188 / 200; 65536 rows in 16, -> 1024 (5 for 16.5) 1024 224 / 211, 512 151 /
        // 148, 256 113 / 116.
        const uint64_t rounds = (on_mean(256u) + cus - 1u) / cus;
        if (A.np > 128u && mean >= 256u && A.nk >= 512u && 11u * rounds * cus <= 4u * on_mean(128u))
            return gather ? launch(k_grouped<T, 256, 256, 2, 4, 2, kPT, kDirect, true, Out>, 256u, 256u, 512u) : launch(k_grouped<T, 256, 256, 2, 4, 2, kPT, kDirect, false, Out>, 256u, 256u, 512u);
        if (by_128) return gather ? launch(k_grouped<T, 128, 128, 2, 2, 2, kPT, kDirect, true, Out>, 128u, 128u, 256u) : launch(k_grouped<T, 128, 128, 2, 2, 2, kPT, kDirect, false, Out>, 128u, 128u, 256u);
        return gather ? launch(k_grouped<T, 64, 64, 2, 2, 4, kPT, kDirect, true, Out>, 64u, 64u, 256u) : launch(k_grouped<T, 64, 64, 2, 2, 4, kPT, kDirect, false, Out>, 64u, 64u, 256u);
    }
}

template <typename T>
hipError_t launch_sums(GatheredOperands A, const Groups& G, float* dw, float* db, Workspace ws, hipStream_t stream) {
    SumOut out{dw, nullptr, 0u, db, A.np, A.nq, A.np % 8u == 0u && aligned(dw, 16u)};
    const uint64_t x_values = (uint64_t)(A.p_count - 1u) * A.ldp + A.np, d_values = (uint64_t)(A.q_count - 1u) * A.ldq + A.nq;
    if (G.rows == 0u || x_values < 8u || d_values < 8u) {
        k_grouped_tiny_sums<T><<<grid_of(((uint64_t)G.count * A.np * A.nq + 255u) / 256u), 256, 0, stream>>>(A, out, G);
        return hipGetLastError();
    }
    const uint64_t length = (uint64_t)A.np * A.nq, bytes = 4u * (length + (db ? A.nq : 0u));
    auto launch = [&](auto kernel, uint32_t bp, uint32_t bq, uint32_t threads) {
        A.tiles_p = ceil_div(A.np, bp);
        A.tiles_q = ceil_div(A.nq, bq);
        const uint64_t tiles = (uint64_t)A.tiles_p * A.tiles_q;
        const uint32_t size  = part_size(G.rows, tiles, device_cu_count(), bytes, ws.bytes), most = G.rows / size + G.count;
        out.parts            = ws.data;
        float* sum_parts     = ws.data + (G.rows / size) * length;
        kernel<<<grid_of(dealt_blocks(most, (uint32_t)tiles)), threads, 0, stream>>>(A, out, G, size, most, sum_parts);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || size >= G.rows) return e;
        return launch_join(G, size, dw, ws.data, length, db, sum_parts, db ? A.nq : 0u, stream);
    };
    const bool gather = A.p_index || A.q_index;
    const bool words  = !whole_chunks(A.p, A.ldp, A.np) || !whole_chunks(A.q, A.ldq, A.nq) || (gather && !(near(A.p_count, A.ldp) && near(A.q_count, A.ldq)));
    // us of a backward pass, sums by tiles of 64 / of 128, fp16: 16384 rows in 16 groups,
    // 256 x 256 (2^30) 30 / 35, 512 x 512 (2^32) 66 / 61; 65536 rows, 256 x 256 (2^32) 82 / 72;
    // by words 255 x 255, 8192 rows 37 / 38, 16384 64 / 54, 65536 188 / 132, 511 x 511, 2048 39 /
    // 43, 4096 55 / 53, 95 x 95, 8192 23 / 28, 32768 41 / 40;
    // 128 / 256: 2048 x 2048, 16384 rows in 8 (2^36) 381 / 409, bf16 4096 x 2048 (2^37) 725 /
    // 688, in 32 groups 965 / 913, 4096 x 4096 (2^38) 1390 / 1239.  Parts enough for one
    // workgroup a CU, for half, one, two and four: 262144 rows in 64 groups 279, 224, 234, 234;
    // 16384 rows in 8 groups, 1024 x 1024, 180, 168, 172, 187.
    const uint64_t work = length * G.rows;
    const bool by_128   = A.np > 64u && A.nq > 64u && work >= (words ? 3ull << 28 : 1ull << 32);
    if (words) return by_128 ? launch(k_grouped_sums<T, 128, 128, 2, 2, kByWords, true>, 128u, 128u, 256u) : launch(k_grouped_sums<T, 64, 64, 2, 2, kByWords, true>, 64u, 64u, 256u);
    if (A.np > 128u && A.nq > 128u && work >= 1ull << 37)
        return gather ? launch(k_grouped_sums<T, 256, 256, 2, 4, kDirect, true>, 256u, 256u, 512u) : launch(k_grouped_sums<T, 256, 256, 2, 4, kDirect, false>, 256u, 256u, 512u);
    if (by_128) return gather ? launch(k_grouped_sums<T, 128, 128, 2, 2, kDirect, true>, 128u, 128u, 256u) : launch(k_grouped_sums<T, 128, 128, 2, 2, kDirect, false>, 128u, 128u, 256u);
    return gather ? launch(k_grouped_sums<T, 64, 64, 2, 2, kDirect, true>, 64u, 64u, 256u) : launch(k_grouped_sums<T, 64, 64, 2, 2, kDirect, false>, 64u, 64u, 256u);
}

template <typename T>
NerfStatus forward(const NerfExtLinearDesc& d, const NerfExtRowGroups& r, const void* x, const void* w, const float* bias, const void* residual, void* y, void* pre, hipStream_t stream) {
    const bool vec = d.out_features % 8u == 0u && d.y_stride % 8u == 0u && aligned(y, 16u) && aligned(pre, 16u) && (!residual || (d.residual_stride % 8u == 0u && aligned(residual, 16u)));
    GatheredOperands A{{w, x, d.in_features, d.x_stride, d.out_features, d.rows, d.in_features, 0u, 0u, 0u}, nullptr, r.x_rows, 0u, r.x_count};
    const RowsForwardOut<T> out{bias, (const T*)residual, y, (T*)pre, d.residual_stride, d.y_stride, d.out_features, d.rows, d.activation, d.out_dtype == NERF_EXT_F32, vec, r.y_rows, r.y_count, nullptr};
    NERF_HIP_TRY((launch_grouped<T, false>(A, out, Groups{r.offsets, r.groups, d.rows}, stream)));
    return NERF_STATUS_OK;
}

template <typename T>
NerfStatus backward(const NerfExtLinearDesc& d, const NerfExtRowGroups& r, const void* x, const void* w, const void* delta, const void* pre, const void* add, void* dx, void* dpre, float* dw, float* db, Workspace ws, hipStream_t stream) {
    const Groups G{r.offsets, r.groups, d.rows};
    if ((dx || dpre) && d.rows) {
        const bool vec = d.in_features % 8u == 0u && (!(add || dx) || d.x_stride % 8u == 0u) && aligned(add, 16u) && aligned(dx, 16u) && aligned(pre, 16u) && aligned(dpre, 16u);
        GatheredOperands A{{w, delta, d.in_features, d.y_stride, d.in_features, d.rows, d.out_features, 0u, 0u, 0u}, nullptr, r.y_rows, 0u, r.y_count};
        const RowsGradientOut<T> out{(const T*)add, (T*)dx, (const T*)pre, (T*)dpre, d.x_stride, d.in_features, d.rows, d.activation, vec, r.x_rows, r.x_count, nullptr};
        NERF_HIP_TRY((launch_grouped<T, true>(A, out, G, stream)));
    }
    if (dw) {
        GatheredOperands A{{x, delta, d.x_stride, d.y_stride, d.in_features, d.out_features, d.rows, 0u, 0u, 0u}, r.x_rows, r.y_rows, r.x_count, r.y_count};
        NERF_HIP_TRY((launch_sums<T>(A, G, dw, db, ws, stream)));
    }
    return NERF_STATUS_OK;
}

}  // namespace

NerfStatus nerf_hip::grouped::check_groups(const NerfExtRowGroups* groups, const NerfExtLinearDesc& d, NerfExtRowGroups& out, const char* fn) {
    auto refuse = [&](const char* why) {
        set_error(std::string(fn) + ": " + why);
        return NERF_STATUS_INVALID_USAGE;
    };
    if (!groups) return refuse("null groups");
    out = *groups;
    if (out.groups == 0u || out.groups > kMaxGroups) return refuse("groups must be 1..4096");
    if (!out.offsets || !aligned(out.offsets, 4u) || !aligned(out.x_rows, 4u) || !aligned(out.y_rows, 4u)) return refuse("null offsets, or an index that is not aligned to its elements");
    if (out.reserved != 0u) return refuse("reserved of the groups must be 0");
    if (out.x_count == 0u) out.x_count = d.rows;
    if (out.y_count == 0u) out.y_count = d.rows;
    if (out.x_count > kMaxRows || out.y_count > kMaxRows) return refuse("more than 2^30 rows");
    if (((uint64_t)d.rows / 64u + out.groups) * ceil_div(std::max(d.in_features, d.out_features), 64u) >= 1ull << 31) return refuse("more than 2^31 tiles of 64 x 64 outputs");
    if ((!out.x_rows && out.x_count != d.rows) || (!out.y_rows && out.y_count != d.rows)) return refuse("x_count and y_count come with x_rows and y_rows");
    return NERF_STATUS_OK;
}

hipError_t nerf_hip::grouped::launch_join(const Groups& G, uint32_t size, float* out, const float* parts, uint64_t length, float* sums, const float* sum_parts, uint32_t sums_length, hipStream_t stream) {
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(ceil_div(length + sums_length, 256u), std::max(1u, 8u * device_cu_count() / G.count));
    k_grouped_join<<<G.count * blocks, 256, 0, stream>>>(G, size, out, parts, length, sums, sum_parts, sums_length, blocks);
    return hipGetLastError();
}

template <typename T, bool kPT>
hipError_t nerf_hip::grouped::launch_ranks(const Groups& G, const T* x, uint64_t ldx, const uint32_t* index, uint32_t count, const T* weight, uint32_t features, uint32_t rank, const float* scales, float* out, hipStream_t stream) {
    GatheredOperands A{{weight, x, kPT ? rank : features, ldx, rank, G.rows, features, 0u, 0u, 0u}, nullptr, index, 0u, count};
    return launch_grouped<T, kPT>(A, PositionOut{out, scales, rank, G.rows, rank % 8u == 0u && aligned(out, 16u), 1.0f}, G, stream);
}
#define NERF_RANKS(T, PT) template hipError_t nerf_hip::grouped::launch_ranks<T, PT>(const Groups&, const T*, uint64_t, const uint32_t*, uint32_t, const T*, uint32_t, uint32_t, const float*, float*, hipStream_t)
NERF_RANKS(half_t, false);
NERF_RANKS(half_t, true);
NERF_RANKS(bf16_t, false);
NERF_RANKS(bf16_t, true);
#undef NERF_RANKS

extern "C" {

NERF_API NerfStatus nerf_ext_grouped_linear_forward(const NerfExtLinearDesc* desc, const NerfExtRowGroups* groups, const void* x, const void* weight, const float* bias, const void* residual, void* y, void* pre, void* workspace,
                                                   uint64_t workspace_bytes, void* stream) {
    NerfExtLinearDesc d;
    NerfExtRowGroups r;
    NerfStatus s = check_desc(desc, d, "nerf_ext_grouped_linear_forward");
    if (s == NERF_STATUS_OK) s = check_groups(groups, d, r, "nerf_ext_grouped_linear_forward");
    if (s != NERF_STATUS_OK) return s;
    (void)workspace_bytes;
    if (d.rows == 0u) return NERF_STATUS_OK;
    NERF_CHECK_ARG(x && weight && y, "nerf_ext_grouped_linear_forward: null x, weight or y");
    NERF_CHECK_ARG(aligned(x, 2u) && aligned(weight, 2u) && aligned(residual, 2u) && aligned(pre, 2u) && aligned(bias, 4u) && aligned(y, d.out_dtype == NERF_EXT_F32 ? 4u : 2u),
                   "nerf_ext_grouped_linear_forward: an array is not aligned to its elements");
    NERF_CHECK_ARG(y != residual || (d.out_dtype == d.dtype && (r.y_count == 1u || d.y_stride == d.residual_stride)), "nerf_ext_grouped_linear_forward: y over residual must have its type and row stride");
    NERF_CHECK_ARG(aligned(workspace, 16u), "nerf_ext_grouped_linear_forward: workspace must be aligned to 16 bytes");
    if (d.dtype == NERF_EXT_F16) return forward<half_t>(d, r, x, weight, bias, residual, y, pre, (hipStream_t)stream);
    return forward<bf16_t>(d, r, x, weight, bias, residual, y, pre, (hipStream_t)stream);
}

NERF_API NerfStatus nerf_ext_grouped_linear_backward(const NerfExtLinearDesc* desc, const NerfExtRowGroups* groups, const void* x, const void* weight, const void* delta, const void* pre, const void* add, void* dx, void* dpre, float* dweight,
                                                    float* dbias, void* workspace, uint64_t workspace_bytes, void* stream) {
    NerfExtLinearDesc d;
    NerfExtRowGroups r;
    NerfStatus s = check_desc(desc, d, "nerf_ext_grouped_linear_backward");
    if (s == NERF_STATUS_OK) s = check_groups(groups, d, r, "nerf_ext_grouped_linear_backward");
    if (s != NERF_STATUS_OK) return s;
    NERF_CHECK_ARG(dx || dpre || dweight, "nerf_ext_grouped_linear_backward: no output");
    NERF_CHECK_ARG(!dbias || dweight, "nerf_ext_grouped_linear_backward: dbias comes with dweight only");
    NERF_CHECK_ARG(d.rows == 0u || delta, "nerf_ext_grouped_linear_backward: null delta");
    NERF_CHECK_ARG(d.rows == 0u || weight || !(dx || dpre), "nerf_ext_grouped_linear_backward: dx and dpre need weight");
    NERF_CHECK_ARG(d.rows == 0u || pre || !dpre, "nerf_ext_grouped_linear_backward: dpre needs pre");
    NERF_CHECK_ARG(d.rows == 0u || x || !dweight, "nerf_ext_grouped_linear_backward: dweight needs x");
    NERF_CHECK_ARG(aligned(x, 2u) && aligned(weight, 2u) && aligned(delta, 2u) && aligned(pre, 2u) && aligned(add, 2u) && aligned(dx, 2u) && aligned(dpre, 2u) && aligned(dweight, 4u) && aligned(dbias, 4u),
                   "nerf_ext_grouped_linear_backward: an array is not aligned to its elements");
    NERF_CHECK_ARG(aligned(workspace, 16u), "nerf_ext_grouped_linear_backward: workspace must be aligned to 16 bytes");
    if (d.rows == 0u && !dweight) return NERF_STATUS_OK;
    const Workspace ws{(float*)workspace, workspace ? workspace_bytes : 0u};
    if (d.dtype == NERF_EXT_F16) return backward<half_t>(d, r, x, weight, delta, pre, add, dx, dpre, dweight, dbias, ws, (hipStream_t)stream);
    return backward<bf16_t>(d, r, x, weight, delta, pre, add, dx, dpre, dweight, dbias, ws, (hipStream_t)stream);
}

}  // extern "C"
