// linear.hip — a linear layer over rows in memory and its gradients
// (include/nerf_ext.h, nerf_ext_linear_*).
//
//   forward:   z = x W^T + b,  y = act(z) + r
//   backward:  g = d W + a,  dx = g,  dpre = g act'(pre),  dW = d^T x,  db = sum d
//
// All three products are one kernel, out(q, p) = sum_k P(p, k) Q(q, k), with
// p the contiguous index of the output:
//   forward  P = W (k contiguous)   Q = x (k contiguous)   k = input feature
//   dx       P = W (p contiguous)   Q = d (k contiguous)   k = output feature
//   dW       P = x (p contiguous)   Q = d (q contiguous)   k = row
// P is the matrix instruction's A operand, so that a lane ends with four
// consecutive p of one q.  An operand whose k is not
// contiguous is read from LDS through the transposing read
// (ds_read_b64_tr_b16), four k of one p a lane, so no operand is transposed in
// memory.  Products are of 16-bit values, exact in 32 bits, and summed in 32
// bits.  The tiles themselves are in linear_device.hpp.
#include "linear_device.hpp"

using namespace nerf_hip;
using namespace nerf_hip::linear;

namespace {

// ----------------------------------------------------------------- product
template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, uint32_t kDepth, bool kPT, bool kQT, Mode kMode, typename Out>
__global__ __launch_bounds__(kWP * kWQ * 64u) void k_product(Operands A, Out out) {
    const uint32_t tile = chip_tile(blockIdx.x, gridDim.x);
    // Where P has more than four tiles, bands of four tiles of Q: the 32 workgroups
    // at work on a chip then share 8 + 4 tiles of the operands, in rows of all of P
    // 16 + 2 (16384 x 4096 -> 4096: 470 us against 478).  With fewer, rows are as
    // square (bands there cost 131072 x 512 -> 512 backward 293 us against 288).
    const uint32_t part = tile / A.tiles_p / A.tiles_q, t = tile - part * A.tiles_p * A.tiles_q, band = A.tiles_p > 4u ? 4u : 1u;
    const uint32_t first = t / (band * A.tiles_p) * band, high = min(band, A.tiles_q - first), in_band = t - first * A.tiles_p;
    const uint32_t tile_p = in_band / high, tile_q = first + in_band % high;
    const uint32_t p0 = tile_p * kBP, q0 = tile_q * kBQ;
    const uint32_t k0 = part * A.k_split, k_end = min(A.nk, k0 + A.k_split);
    if constexpr (std::is_same_v<Out, SumOut>) {
        if (part) out.out = out.parts + (part - 1u) * out.part;
        if (out.row_sums) out.row_sums += (uint64_t)part * out.nq;
    }
    product<T, kBP, kBQ, kWP, kWQ, kDepth, kPT, kQT, kMode>(A, out, Place{p0, q0, k0, k_end, 0u, 0u});
}

// ------------------------------------------------------------ short sums
// Many rows and at most 32 kKS <= 256 k: memory bound.  A wave keeps its
// 16 kFP p of P in registers for all k (at most 128 of them) and goes through
// the rows 16 at a time: it reads Q as the matrix instruction takes it, straight
// from memory, the next rows' Q and epilogue inputs being on their way while
// these rows' outputs leave.  Waves do not wait for each other.  Waves of a
// workgroup that hold other p read the same Q at about the same time, from the
// CU's cache.  262144 x 256 -> 256 with residual and pre takes 109 us = 4.9 TB/s, a
// copy's rate (by tiles 130); its input gradient 129.
template <typename T, uint32_t kKS, uint32_t kFP, bool kPT, bool kRagged, bool kWords, typename Out>
__global__ __launch_bounds__(kStreamWaves * 64u) void k_stream(Operands A, Out out, uint32_t p_waves) {
    // Where P takes half of the registers, the outputs' edges have to do without any.
    if constexpr (kKS * kFP == 32u) out.vec = true;
    constexpr uint32_t kSP = 16u * kFP, kBP = 256u;
    constexpr uint32_t kLanes = kSP / 8u, kPasses = 16u * kLanes / 64u;
    using x8 = typename Vec<T>::x8;
    __shared__ uint4 lds[kBP * 8u];
    __shared__ floatx4 lds_bias[Out::kBias ? kBP / 4u : 1u];
    static_assert(kStreamWaves * kSP * 4u <= kBP * 8u);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t wp = wave % p_waves * kSP, p0 = blockIdx.y * p_waves * kSP;

    x8 fp[kKS][kFP];
    hold_weights<T, kBP, kPT>(A, out, p0, wp, lds, lds_bias, fp);

    // Rows: lane l has k 8 (l / 16) + 0..7 of every 32 of row l % 16.
    const uint32_t groups = kStreamWaves / p_waves, tiles = (A.nq + 15u) / 16u, stride = gridDim.x * groups;
    const uint32_t l = lane & 15u, g = lane >> 4;
    const uint32_t whole = A.nk / 32u;  // steps of 32 k that every row has in full
    // kRagged, the step after them: `some` of the lane's 8 k are left.  They are
    // fetched as 8 values that end with the row (or begin with the array, in its
    // first rows), and moved down by `down` values when they are used.
    const uint32_t left = A.nk % 32u, some = left > 8u * g ? min(8u, left - 8u * g) : 0u;
    // What is on its way: the Q and the epilogue inputs of the kAhead next tiles of
    // rows, as many as the registers hold beside P.  (With one, 100003 x 64 -> 256
    // took 33 us from memory and 24 us from cache.)
    constexpr uint32_t kAhead = kKS <= 2u ? 3u : kKS * kFP < 16u || (kKS * kFP == 16u && !kWords && sizeof(typename Out::Aux) <= 16u) ? 2u : 1u;
    // Where even one tile's epilogue inputs take more registers than there are
    // beside this tile's, they are fetched in their place as these are used.
    constexpr bool kLate = kKS * kFP == 32u && sizeof(typename Out::Aux) > 16u;
    struct Coming {
        Eight<kWords> q[kKS];
        uint32_t down, place, place_last;  // place: see Eight::value
        typename Out::Aux aux[kPasses];
    };
    Coming coming[kAhead];
    const uint32_t row = lane / kLanes, col = 8u * (lane % kLanes), p = p0 + wp + col;
    const uint32_t n = p < out.np ? min(8u, out.np - p) : 0u;
    auto inside = [&](uint32_t tile, uint32_t pass) { return tile < tiles && tile * 16u + (64u / kLanes) * pass + row < out.nq ? n : 0u; };
    auto fetch_q = [&](Coming& c, uint32_t tile) {
        const uint64_t first = (uint64_t)min(tile * 16u + l, A.nq - 1u) * A.ldq + 8u * g;
        const T* at          = (const T*)A.q + first;
        c.place              = value_number(at);
#pragma unroll
        for (uint32_t s = 0; s < kKS; ++s) {
            if (s < whole) c.q[s].fetch(at + 32u * s);
            if (kRagged && s == whole) {
                const uint64_t end = first + 32u * s + some, from = end > 8u ? end - 8u : 0ull;
                c.down             = some ? (uint32_t)(first + 32u * s - from) : 0u;
                const T* at_last   = (const T*)A.q + (some ? from : 0ull);
                c.place_last       = value_number(at_last);
                c.q[s].fetch(at_last);
            }
        }
    };
    auto fetch_aux = [&](Coming& c, uint32_t tile, uint32_t t) { c.aux[t] = out.load(tile * 16u, (64u / kLanes) * t + row, p, inside(tile, t)); };
    floatx4* strip = reinterpret_cast<floatx4*>(lds) + wave * (kSP * 4u);
    const uint32_t first_tile = __builtin_amdgcn_readfirstlane(blockIdx.x * groups + wave / p_waves);
#pragma unroll
    for (uint32_t d = 0; d < kAhead; ++d) {
#pragma unroll
        for (uint32_t s = 0; s < kKS; ++s) coming[d].q[s] = Eight<kWords>{};
        if (first_tile + d * stride < tiles) {
            fetch_q(coming[d], first_tile + d * stride);
#pragma unroll
            for (uint32_t t = 0; t < kPasses; ++t) fetch_aux(coming[d], first_tile + d * stride, t);
        }
    }
    for (uint32_t turn = first_tile; turn < tiles; turn += kAhead * stride) {
#pragma unroll
        for (uint32_t d = 0; d < kAhead; ++d) {
            const uint32_t tile = turn + d * stride, later = tile + kAhead * stride;
            Coming& c           = coming[d];
            if (tile < tiles) {
                floatx4 acc[kFP];
#pragma unroll
                for (uint32_t i = 0; i < kFP; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t s = 0; s < kKS; ++s) {
                    uint4 v = c.q[s].value(c.place);
                    if (kRagged && s == whole) v = settled(c.q[s].value(c.place_last), c.down, some);
#pragma unroll
                    for (uint32_t i = 0; i < kFP; ++i) acc[i] = Vec<T>::mfma(fp[s][i], __builtin_bit_cast(x8, v), acc[i]);
                }
                typename Out::Aux aux[kPasses];
#pragma unroll
                for (uint32_t t = 0; t < kPasses; ++t) aux[t] = c.aux[t];
                if (later < tiles) {
                    fetch_q(c, later);
#pragma unroll
                    for (uint32_t t = 0; t < kPasses; ++t)
                        if (!kLate) fetch_aux(c, later, t);
                }
#pragma unroll
                for (uint32_t i = 0; i < kFP; ++i) strip[l * (kSP / 4u) + ((4u * i + g) ^ (l & 7u))] = acc[i];
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
                for (uint32_t t = 0; t < kPasses; ++t) {
                    const uint32_t r = (64u / kLanes) * t + row;
                    floatx8 v;
                    v.lo = strip[r * (kSP / 4u) + ((col / 4u) ^ (r & 7u))];
                    v.hi = strip[r * (kSP / 4u) + ((col / 4u + 1u) ^ (r & 7u))];
                    out.put(tile * 16u, r, p, inside(tile, t), v, bias8<Out>(reinterpret_cast<const float*>(lds_bias), wp + col), aux[t]);
                    if (kLate) fetch_aux(c, later, t);
                }
                asm volatile("" ::: "memory");
            }
        }
    }
}

template <typename T, uint32_t kF, bool kWords>
__global__ __launch_bounds__(kFewWaves * 64u) void k_few_forward(Operands A, ForwardOut<T> out) {
    __shared__ floatx4 lds[few_lds(kF, kF) / 16u];
    few_tile<T, kF, kF, false, false, kWords>(A, out, Place{blockIdx.x * 16u * kF, blockIdx.y * 16u * kF, 0u, A.nk, 0u, 0u}, reinterpret_cast<char*>(lds), nullptr);
}

// Both gradients in one launch: first the tiles of dx, x_tiles across and
// x_blocks in all, then those of dW.
template <typename T, uint32_t kF, bool kWords>
__global__ __launch_bounds__(kFewWaves * 64u) void k_few_backward(Operands X, InputGradientOut<T> x_out, uint32_t x_tiles, uint32_t x_blocks, Operands W, SumOut w_out, uint32_t w_tiles) {
    __shared__ floatx4 lds[few_lds(kF, kF) / 16u];
    __shared__ float lds_sums[kFewWaves * 16u * kF];
    if (blockIdx.x < x_blocks) {
        few_tile<T, kF, kF, true, false, kWords>(X, x_out, Place{blockIdx.x % x_tiles * 16u * kF, blockIdx.x / x_tiles * 16u * kF, 0u, X.nk, 0u, 0u}, reinterpret_cast<char*>(lds), nullptr);
    } else {
        const uint32_t b = blockIdx.x - x_blocks;
        few_tile<T, kF, kF, true, true, kWords>(W, w_out, Place{b % w_tiles * 16u * kF, b / w_tiles * 16u * kF, 0u, W.nk, 0u, 0u}, reinterpret_cast<char*>(lds), lds_sums);
    }
}

// Operands of fewer than eight values in all (at most eight k then): a thread
// computes eight outputs from memory.
template <typename T, bool kPT, bool kQT, typename Out>
__global__ __launch_bounds__(256) void k_tiny(Operands A, Out out) {
    const uint32_t eights = (out.np + 7u) / 8u;
    const uint64_t total = (uint64_t)eights * out.nq;
    for (uint64_t base = (uint64_t)blockIdx.x * 256u; base < total; base += (uint64_t)gridDim.x * 256u) {
        const uint64_t at = base + threadIdx.x;
        const uint32_t q0 = (uint32_t)(base / eights), q = (uint32_t)(at / eights), p = 8u * (uint32_t)(at % eights), n = at < total ? min(8u, out.np - p) : 0u;
        const typename Out::Aux aux = out.load(q0, q - q0, p, n);
        floatx8 v = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, b = v;
        float sum = 0.0f;
        for (uint32_t k = 0; n && k < A.nk; ++k) {
            const float x = (float)((const T*)A.q)[kQT ? k * A.ldq + q : q * A.ldq + k];
            sum += x;
#pragma unroll
            for (uint32_t r = 0; r < 8u; ++r) v[r] += r < n ? x * (float)((const T*)A.p)[kPT ? k * A.ldp + p + r : (uint64_t)(p + r) * A.ldp + k] : 0.0f;
        }
        if constexpr (Out::kBias) {
            if (out.bias) {
#pragma unroll
                for (uint32_t r = 0; r < 8u; ++r) b[r] = r < n ? out.bias[p + r] : 0.0f;
            }
        }
        out.put(q0, q - q0, p, n, v, b, aux);
        if constexpr (std::is_same_v<Out, SumOut>) {
            if (out.row_sums && n && p == 0u) out.row_sums[q] = sum;
        }
    }
}

// Joins the parts of a sum that was split over k: kSlices slices of a workgroup
// take every kSlices-th part each, in order, and the slices are added in theirs,
// so the result is the same every time.  (With one thread an output the reads of
// 128 parts of 256 x 256 sums, one after another, took 73 us; with 16 slices for
// two parts of 4096 x 2048 sums, 14 of them idle, 59 us where one takes 19 us.)
template <uint32_t kSlices, typename Out>
__global__ __launch_bounds__(256) void k_join(const float* first_part, const float* __restrict__ parts, uint64_t part, uint32_t count, const float* __restrict__ sums, float* __restrict__ row_sums, Out out) {
    constexpr uint32_t kJoined = 256u / kSlices;
    __shared__ floatx4 slice_sum[2][kSlices][kJoined];
    const uint32_t eights = (out.np + 7u) / 8u, slice = threadIdx.x / kJoined, mine = threadIdx.x % kJoined;
    const uint64_t total = (uint64_t)eights * out.nq;
    const bool vec = out.np % 8u == 0u && ((uintptr_t)first_part & 15u) == 0u;
    for (uint64_t base = (uint64_t)blockIdx.x * kJoined; base < total; base += (uint64_t)gridDim.x * kJoined) {
        const uint64_t at = base + mine;
        const uint32_t q = (uint32_t)(at / eights), p = 8u * (uint32_t)(at % eights), n = at < total ? min(8u, out.np - p) : 0u;
        // The epilogues count rows from a uniform one: the workgroup's first.
        const uint32_t q0 = (uint32_t)(base / eights);
        const typename Out::Aux aux = out.load(q0, q - q0, p, slice == 0u ? n : 0u);
        floatx8 v = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (n) {
#pragma unroll 8
            for (uint32_t c = slice; c < count; c += kSlices) {
                const float* src = (c ? parts + (c - 1u) * part : first_part) + (uint64_t)q * out.np + p;
                if (vec) {
                    v.lo += reinterpret_cast<const floatx4*>(src)[0];
                    v.hi += reinterpret_cast<const floatx4*>(src)[1];
                } else {
#pragma unroll
                    for (uint32_t r = 0; r < 8u; ++r) v[r] += r < n ? src[r] : 0.0f;
                }
            }
        }
        if constexpr (kSlices > 1u) {
            __syncthreads();
            slice_sum[0][slice][mine] = v.lo;
            slice_sum[1][slice][mine] = v.hi;
            __syncthreads();
        }
        if (slice == 0u) {
#pragma unroll
            for (uint32_t c = 1; c < kSlices; ++c) {
                v.lo += slice_sum[0][c][mine];
                v.hi += slice_sum[1][c][mine];
            }
            floatx8 b = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (Out::kBias) {
                if (out.bias) {
#pragma unroll
                    for (uint32_t r = 0; r < 8u; ++r) b[r] = r < n ? out.bias[p + r] : 0.0f;
                }
            }
            out.put(q0, q - q0, p, n, v, b, aux);
        }
    }
    if (row_sums) {
        float(*sum)[kJoined] = reinterpret_cast<float(*)[kJoined]>(slice_sum);
        for (uint32_t base = blockIdx.x * kJoined; base < out.nq; base += gridDim.x * kJoined) {
            const uint32_t q = base + mine;
            float s = 0.0f;
            if (q < out.nq) {
#pragma unroll 8
                for (uint32_t c = slice; c < count; c += kSlices) s += sums[(uint64_t)c * out.nq + q];
            }
            __syncthreads();
            sum[slice][mine] = s;
            __syncthreads();
            if (slice == 0u && q < out.nq) {
#pragma unroll
                for (uint32_t c = 1; c < kSlices; ++c) s += sum[c][mine];
                row_sums[q] = s;
            }
        }
    }
}

// ------------------------------------------------------------------- host

template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, uint32_t kDepth, bool kPT, bool kQT, Mode kMode, bool kSplit = true, typename Out>
hipError_t launch_tiles(Operands A, Out out, float* row_sums, Workspace ws, hipStream_t stream) {
    const uint32_t tp = ceil_div(A.np, kBP), tq = ceil_div(A.nq, kBQ);
    // Split over k until every CU has its workgroups (two; one of the widest
    // tile, whose buffers take the LDS of a CU), with four tiles of k a part at
    // least, as far as the workspace holds the parts.  Outputs of 16 bits are split
    // in four at least and from 1024 k on, where the parts' way through memory
    // pays: 16 x 8192 -> 2048 12 us (whole 31), 1024 x 1024 -> 1024 14.5 in two
    // parts and 8.6 whole, 512 x 1024 -> 1024 11.4 in four and 7.9 whole.
    // The first part of a plain sum is kept where the sum will be.
    const uint64_t part = (uint64_t)A.np * A.nq, words = ws.bytes / 4u;
    constexpr bool kSums = std::is_same_v<Out, SumOut>;
    const uint64_t held = kSums ? (words + part) / (part + (row_sums ? A.nq : 0u)) : words / part;
    const uint64_t fill = (kBP == 256u ? 1u : 2u) * device_cu_count();
    uint64_t splits = kSplit ? fill / ((uint64_t)tp * tq) : 1u;
    splits = std::min<uint64_t>({splits, ceil_div(A.nk, 4u * kBK), held});
    if (splits <= 1u || (!kSums && (splits < 4u || A.nk <= 1024u))) splits = 1u;
    A.k_split = ceil_div(ceil_div(A.nk, kBK), splits) * kBK;
    if (A.k_split == 0u) A.k_split = kBK;
    const uint32_t parts = std::max(1u, ceil_div(A.nk, A.k_split));
    A.tiles_p           = tp;
    A.tiles_q           = tq;
    const uint32_t grid = tp * tq * parts;
    constexpr uint32_t kThreads = kWP * kWQ * 64u;
    if constexpr (kSplit) {
        if (parts > 1u) {
            SumOut so{};
            float* rest = ws.data;
            if constexpr (kSums) {
                so = out;
            } else {
                so.out = ws.data;
                so.np  = A.np;
                so.nq  = A.nq;
                so.vec = A.np % 8u == 0u;
                rest += part;
            }
            so.parts    = rest;
            so.part     = part;
            float* sums = row_sums ? rest + (parts - 1u) * part : nullptr;
            so.row_sums = sums;
            k_product<T, kBP, kBQ, kWP, kWQ, kDepth, kPT, kQT, kMode, SumOut><<<grid, kThreads, 0, stream>>>(A, so);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            const uint64_t eights = (uint64_t)ceil_div(A.np, 8u) * A.nq;
            auto join = [&](auto slices) { k_join<slices(), Out><<<(uint32_t)std::min<uint64_t>(ceil_div(eights, 256u / slices()), 4096u), 256, 0, stream>>>(so.out, rest, part, parts, sums, row_sums, out); };
            // 16-bit outputs have four parts at least: four splits or more of at least
            // 17 tiles of k make as many.
            if (parts >= 16u) join(std::integral_constant<uint32_t, 16u>{});
            else if (!kSums || parts >= 4u) join(std::integral_constant<uint32_t, 4u>{});
            else if constexpr (kSums) join(std::integral_constant<uint32_t, 1u>{});
            return hipGetLastError();
        }
    }
    k_product<T, kBP, kBQ, kWP, kWQ, kDepth, kPT, kQT, kMode, Out><<<grid, kThreads, 0, stream>>>(A, out);
    return hipGetLastError();
}

// Whether an operand has fewer than eight values from its first to its last.
bool few_values(const Operands& A, bool pt, bool qt) {
    auto values = [](uint64_t ld, uint32_t n, uint32_t nk, bool t) { return t ? (uint64_t)(nk - 1u) * ld + n : (uint64_t)(n - 1u) * ld + nk; };
    return A.nk == 0u || values(A.ldp, A.np, A.nk, pt) < 8u || values(A.ldq, A.nq, A.nk, qt) < 8u;
}

template <typename T, uint32_t kKS, bool kPT, typename Out>
hipError_t launch_stream(const Operands& A, const Out& out, hipStream_t stream) {
    // p a wave holds: 64, whose 16-bit outputs are whole lines; 32 where there are
    // no more.
    const bool ragged = A.nk % 32u != 0u, odd = odd_rows(A.q, A.ldq), narrow = A.np <= 32u;
    const uint32_t wide = narrow ? 32u : 64u, most = 256u / wide;
    uint32_t p_waves = 1u;
    while (p_waves < most && wide * p_waves < A.np) p_waves *= 2u;
    const uint32_t across = ceil_div(A.np, wide * p_waves), tiles = ceil_div(A.nq, 16u), groups = kStreamWaves / p_waves;
    // One workgroup fills a CU's registers; every one goes through as many rows.
    const dim3 grid(std::min(ceil_div(tiles, groups), std::max(1u, device_cu_count() / across)), across);
    constexpr uint32_t kThreads = kStreamWaves * 64u;
    auto launch = [&](auto p, auto cut, auto words) { k_stream<T, kKS, p(), kPT, cut(), words(), Out><<<grid, kThreads, 0, stream>>>(A, out, p_waves); };
    auto by_width = [&](auto cut, auto words) {
        if (narrow) launch(std::integral_constant<uint32_t, 2u>{}, cut, words);
        else launch(std::integral_constant<uint32_t, 4u>{}, cut, words);
    };
    if constexpr (kKS <= 2u) {
        if (odd) {
            by_width(std::true_type{}, std::true_type{});
            return hipGetLastError();
        }
        if (ragged) {
            by_width(std::true_type{}, std::false_type{});
            return hipGetLastError();
        }
    }
    by_width(std::false_type{}, std::false_type{});
    return hipGetLastError();
}

// Whether the streamed kernel takes a product, by steps of 32 k (at most 8): with
// so many rows that its start, a CU's weights, is small beside them, and beyond
// two steps only where rows and outputs are whole; what cut ones need then takes
// the registers of rows on their way.  Streamed against by tiles, in us: 262144
// rows, 256 -> 256 with residual 116 / 130, and 65536 without 34 / 30; 128 -> 256,
// 131072 rows 43 / 48 and 32768 rows 13 / 11; 64 -> 256, 65536 rows 17 / 19 and
// 32768 rows 11.8 / 11.3; 32 -> 64, 131072 rows 11 / 17.  Cut: 262144 x 240 ->
// 256 141 / 113, 100 -> 250 126 / 99, 256 -> 250 206 / 119; 65536 x 63 -> 255
// 24 / 25.  Beyond 1024 p, 65536 x 256 -> 2048 211 / 192.  Input gradients move
// more beside the product and come to it with fewer rows: 65536 x 256 -> 256
// backward 69 / 79.
bool streamed(const Operands& A, bool vec, bool gradient) {
    const uint32_t steps = A.nk <= 32u ? 1u : A.nk <= 64u ? 2u : A.nk <= 128u ? 4u : 8u;
    if (A.nk > 256u || A.np > 1024u || A.nq < 16384u * (gradient ? (steps + 1u) / 2u : steps)) return false;
    return steps <= 2u || (A.nk % 32u == 0u && vec && !odd_rows(A.q, A.ldq));
}

template <typename T, bool kPT, bool kQT, typename Out>
hipError_t launch_product(Operands A, Out out, float* row_sums, Workspace ws, hipStream_t stream) {
    if (few_values(A, kPT, kQT)) {
        const uint64_t threads = (uint64_t)ceil_div(A.np, 8u) * A.nq;
        k_tiny<T, kPT, kQT, Out><<<(uint32_t)std::min<uint64_t>(ceil_div(threads, 256u), 8u * device_cu_count()), 256, 0, stream>>>(A, out);
        return hipGetLastError();
    }
    if constexpr (!kQT) {
        if (streamed(A, out.vec, kPT)) {
            if (A.nk <= 32u) return launch_stream<T, 1u, kPT>(A, out, stream);
            if (A.nk <= 64u) return launch_stream<T, 2u, kPT>(A, out, stream);
            if (A.nk <= 128u) return launch_stream<T, 4u, kPT>(A, out, stream);
            return launch_stream<T, 8u, kPT>(A, out, stream);
        }
    }
    // The tile.  Larger ones read less, smaller ones occupy the card with fewer
    // outputs.  In us, by tiles of 64 / 128 / 256:
    //   16-bit outputs by their tiles' number: 128 from 7/8 of the CUs on, 256 from
    //   as many as CUs.  2048 x 1024 -> 1024 13 / 19 / -, 3000 x 1200 -> 1200
    //   26 / 23 / -, 8192 x 1024 -> 1024 37 / 24 / 37, 16384 x 1024 -> 1024
    //   82 / 56 / 49, 16384 x 4096 -> 4096 - / - / 470.  Of less than 512 k the
    //   largest have too few steps.
    //   Gradients of weights, whose k is split until the card is full, by the work:
    //   128 from 2^32 products on, 256 from 2^35.  65536 x 128 -> 128 (2^30)
    //   16 / 21 / -, with dx 37 / 43 / -; 65536 x 256 -> 256 (2^32) with dx
    //   76 / 69 / -, 32768 x 512 -> 512 (2^33) 36 / 38 / 46, 8192 x 1024 -> 1024 (2^33) 36 / 32 / 43, 262144 x 256 -> 256
    //   (2^34) 97 / 77 / 96, 131072 x 512 -> 512 (2^35) 164 / 107 / 102,
    //   16384 x 2048 -> 2048 (2^36) 324 / 165 / 153.
    // Of the larger tiles only those of weights' gradients (kLong) are split: 16-bit
    // outputs get them where they are too many for a split in four.
    constexpr bool kLong = kPT && kQT;
    const uint64_t cus  = device_cu_count(), work = (uint64_t)A.np * A.nq * A.nk;
    auto tiles          = [&](uint32_t b) { return (uint64_t)ceil_div(A.np, b) * ceil_div(A.nq, b); };
    const bool by_128   = A.np > 64u && A.nq > 64u && (kLong ? work >= 1ull << 32 : 8u * tiles(128u) >= 7u * cus);
    if (!whole_chunks(A.p, A.ldp, kPT ? A.np : A.nk) || !whole_chunks(A.q, A.ldq, kQT ? A.nq : A.nk)) {
        // Rows on their way as words, two tiles (86 us for 20011 x 1209 -> 487; with
        // one 93); as chunks one (68 us for 20011 x 1210 -> 488, with two 75).
        const bool odd = odd_rows(A.p, A.ldp) || odd_rows(A.q, A.ldq);
        if (by_128) return odd ? launch_tiles<T, 128, 128, 2, 2, 3, kPT, kQT, kByWords, kLong>(A, out, row_sums, ws, stream) : launch_tiles<T, 128, 128, 2, 2, 2, kPT, kQT, kByChunks, kLong>(A, out, row_sums, ws, stream);
        return odd ? launch_tiles<T, 64, 64, 2, 2, 4, kPT, kQT, kByWords>(A, out, row_sums, ws, stream) : launch_tiles<T, 64, 64, 2, 2, 4, kPT, kQT, kByChunks>(A, out, row_sums, ws, stream);
    }
    if (A.np > 128u && A.nq > 128u && A.nk >= 512u && (kLong ? work >= 1ull << 35 : tiles(256u) >= cus))
        return launch_tiles<T, 256, 256, 2, 4, 2, kPT, kQT, kDirect, kLong>(A, out, row_sums, ws, stream);
    if (by_128) return launch_tiles<T, 128, 128, 2, 2, 2, kPT, kQT, kDirect, kLong>(A, out, row_sums, ws, stream);
    return launch_tiles<T, 64, 64, 2, 2, 4, kPT, kQT, kDirect>(A, out, row_sums, ws, stream);
}

// Products of few tiles are those of at most 4096 k (1 x 4096 -> 4096 9 us, by
// larger tiles with k split over workgroups 13; 1 x 8192 -> 4096 17.5 against
// 15.5) with at most two tiles a CU.
bool few_operands(const Operands& A, bool pt, bool qt) { return A.nk <= kFewMaxK && !few_values(A, pt, qt); }
uint64_t few_tiles(const Operands& A, uint32_t f) { return (uint64_t)ceil_div(A.np, 16u * f) * ceil_div(A.nq, 16u * f); }

// rows beyond gridDim's range of 64-row tiles are taken in launches of this many.
constexpr uint32_t kRowsPerLaunch = 65535u * 64u;

template <typename T>
NerfStatus forward(const NerfExtLinearDesc& d, const void* x, const void* w, const float* bias, const void* residual, void* y, void* pre, Workspace ws, hipStream_t stream) {
    const bool y32 = d.out_dtype == NERF_EXT_F32;
    const bool vec = d.out_features % 8u == 0u && d.y_stride % 8u == 0u && aligned(y, 16u) && aligned(pre, 16u) && (!residual || (d.residual_stride % 8u == 0u && aligned(residual, 16u)));
    const Operands all{w, x, d.in_features, d.x_stride, d.out_features, d.rows, d.in_features, 0u, 0u, 0u};
    if (few_operands(all, false, false)) {
        const ForwardOut<T> out{bias, (const T*)residual, y, (T*)pre, d.residual_stride, d.y_stride, d.out_features, d.rows, d.activation, y32, vec};
        // Tiles of 16 outputs a side up to two a CU; of 32 one (512 x 1024 -> 1024,
        // two: 11 us, by tiles of 64 8) and with odd rows two (353 x 1115 -> 705 13.2
        // us, by tiles of 64 14.7).
        const uint32_t cus = device_cu_count();
        const bool odd     = odd_rows(x, d.x_stride) || odd_rows(w, d.in_features);
        auto launch        = [&](auto f) {
            const dim3 grid(ceil_div(all.np, 16u * f()), ceil_div(all.nq, 16u * f()));
            if (odd) k_few_forward<T, f(), true><<<grid, kFewWaves * 64u, 0, stream>>>(all, out);
            else k_few_forward<T, f(), false><<<grid, kFewWaves * 64u, 0, stream>>>(all, out);
            NERF_LAUNCH_CHECK("k_few_forward");
            return NERF_STATUS_OK;
        };
        if (few_tiles(all, 1u) <= 2u * cus) return launch(std::integral_constant<uint32_t, 1u>{});
        if (few_tiles(all, 2u) <= (odd ? 2u : 1u) * cus) return launch(std::integral_constant<uint32_t, 2u>{});
    }
    for (uint64_t r0 = 0; r0 < d.rows; r0 += kRowsPerLaunch) {
        const uint32_t n = (uint32_t)std::min<uint64_t>(kRowsPerLaunch, d.rows - r0);
        const Operands A{w, (const T*)x + r0 * d.x_stride, d.in_features, d.x_stride, d.out_features, n, d.in_features, 0u, 0u, 0u};
        void* yo = y32 ? (void*)((float*)y + r0 * d.y_stride) : (void*)((T*)y + r0 * d.y_stride);
        const ForwardOut<T> out{bias, residual ? (const T*)residual + r0 * d.residual_stride : nullptr, yo, pre ? (T*)pre + r0 * d.out_features : nullptr, d.residual_stride, d.y_stride, d.out_features, n, d.activation, y32, vec};
        NERF_HIP_TRY((launch_product<T, false, false>(A, out, nullptr, ws, stream)));
    }
    return NERF_STATUS_OK;
}

template <typename T>
NerfStatus backward(const NerfExtLinearDesc& d, const void* x, const void* w, const void* delta, const void* pre, const void* add, void* dx, void* dpre, float* dw, float* db, Workspace ws, hipStream_t stream) {
    const bool vec = d.in_features % 8u == 0u && (!(add || dx) || d.x_stride % 8u == 0u) && aligned(add, 16u) && aligned(dx, 16u) && aligned(pre, 16u) && aligned(dpre, 16u);
    const Operands all_x{w, delta, d.in_features, d.y_stride, d.in_features, d.rows, d.out_features, 0u}, all_w{x, delta, d.x_stride, d.y_stride, d.in_features, d.out_features, d.rows, 0u, 0u, 0u};
    const SumOut w_out{dw, nullptr, 0u, db, d.in_features, d.out_features, d.in_features % 8u == 0u && aligned(dw, 16u)};
    const bool to_x = (dx || dpre) && d.rows != 0u;
    if ((!to_x || few_operands(all_x, true, false)) && (!dw || few_operands(all_w, true, true))) {
        const InputGradientOut<T> x_out{(const T*)add, (T*)dx, (const T*)pre, (T*)dpre, d.x_stride, d.in_features, d.rows, d.activation, vec};
        // The smallest tile with at most two workgroups a CU.  Those of 16 and 32 a side
        // run at once; those of 64, whose 130 KB of LDS leave a CU room for one, run in
        // up to two turns, and are taken up to 2048 rows, which a workgroup of dW goes
        // through (2048 x 256 -> 256 11 us and 15 in three launches, 1024 x 1024 -> 1024,
        // 512 of them, 18 and 21, but 4096 x 256 -> 256 23 and 17).
        const uint32_t most = 2u * device_cu_count();
        auto blocks         = [&](uint32_t f) { return (to_x ? few_tiles(all_x, f) : 0u) + (dw ? few_tiles(all_w, f) : 0u); };
        auto launch         = [&](auto f) {
            const uint32_t across = ceil_div(d.in_features, 16u * f());
            const uint32_t x_blocks = to_x ? (uint32_t)few_tiles(all_x, f()) : 0u, grid = (uint32_t)blocks(f());
            if (odd_rows(x, d.x_stride) || odd_rows(w, d.in_features) || odd_rows(delta, d.y_stride)) k_few_backward<T, f(), true><<<grid, kFewWaves * 64u, 0, stream>>>(all_x, x_out, across, x_blocks, all_w, w_out, across);
            else k_few_backward<T, f(), false><<<grid, kFewWaves * 64u, 0, stream>>>(all_x, x_out, across, x_blocks, all_w, w_out, across);
            NERF_LAUNCH_CHECK("k_few_backward");
            return NERF_STATUS_OK;
        };
        if (blocks(1u) <= most) return launch(std::integral_constant<uint32_t, 1u>{});
        if (blocks(2u) <= most) return launch(std::integral_constant<uint32_t, 2u>{});
        if (d.rows <= 2048u && blocks(4u) <= most) return launch(std::integral_constant<uint32_t, 4u>{});
    }
    if (to_x) {
        for (uint64_t r0 = 0; r0 < d.rows; r0 += kRowsPerLaunch) {
            const uint32_t n = (uint32_t)std::min<uint64_t>(kRowsPerLaunch, d.rows - r0);
            const Operands A{w, (const T*)delta + r0 * d.y_stride, d.in_features, d.y_stride, d.in_features, n, d.out_features, 0u, 0u, 0u};
            const InputGradientOut<T> out{add ? (const T*)add + r0 * d.x_stride : nullptr, dx ? (T*)dx + r0 * d.x_stride : nullptr, pre ? (const T*)pre + r0 * d.in_features : nullptr,
                                          dpre ? (T*)dpre + r0 * d.in_features : nullptr, d.x_stride, d.in_features, n, d.activation, vec};
            NERF_HIP_TRY((launch_product<T, true, false>(A, out, nullptr, ws, stream)));
        }
    }
    if (dw) NERF_HIP_TRY((launch_product<T, true, true>(all_w, w_out, db, ws, stream)));
    return NERF_STATUS_OK;
}

}  // namespace

NerfStatus nerf_hip::linear::check_desc(const NerfExtLinearDesc* desc, NerfExtLinearDesc& d, const char* fn) {
    auto refuse = [&](const char* why) {
        set_error(std::string(fn) + ": " + why);
        return NERF_STATUS_INVALID_USAGE;
    };
    if (!desc) return refuse("null descriptor");
    d = *desc;
    if (d.rows > kMaxRows) return refuse("more than 2^30 rows");
    if (d.in_features == 0u || d.in_features > kMaxFeatures || d.out_features == 0u || d.out_features > kMaxFeatures) return refuse("features must be 1..65536");
    if (d.dtype != NERF_EXT_F16 && d.dtype != NERF_EXT_BF16) return refuse("dtype must be NERF_EXT_F16 or NERF_EXT_BF16");
    if (d.out_dtype != d.dtype && d.out_dtype != NERF_EXT_F32) return refuse("out_dtype must be dtype or NERF_EXT_F32");
    if (d.activation > NERF_EXT_ACT_GELU) return refuse("unknown activation");
    if (d.reserved != 0u) return refuse("reserved must be 0");
    if (d.x_stride == 0u) d.x_stride = d.in_features;
    if (d.y_stride == 0u) d.y_stride = d.out_features;
    if (d.residual_stride == 0u) d.residual_stride = d.out_features;
    if (d.x_stride < d.in_features || d.y_stride < d.out_features || d.residual_stride < d.out_features) return refuse("a row stride is smaller than the row");
    if (d.x_stride > kMaxStride || d.y_stride > kMaxStride || d.residual_stride > kMaxStride) return refuse("a row stride is above 2^20");
    return NERF_STATUS_OK;
}

extern "C" {

NERF_API NerfStatus nerf_ext_linear_forward(const NerfExtLinearDesc* desc, const void* x, const void* weight, const float* bias, const void* residual, void* y, void* pre, void* workspace, uint64_t workspace_bytes, void* stream) {
    NerfExtLinearDesc d;
    const NerfStatus s = check_desc(desc, d, "nerf_ext_linear_forward");
    if (s != NERF_STATUS_OK) return s;
    if (d.rows == 0u) return NERF_STATUS_OK;
    NERF_CHECK_ARG(x && weight && y, "nerf_ext_linear_forward: null x, weight or y");
    NERF_CHECK_ARG(aligned(x, 2u) && aligned(weight, 2u) && aligned(residual, 2u) && aligned(pre, 2u) && aligned(bias, 4u) && aligned(y, d.out_dtype == NERF_EXT_F32 ? 4u : 2u), "nerf_ext_linear_forward: an array is not aligned to its elements");
    // A lane reads the residuals of the outputs that it writes, so y may take their
    // place; laid out otherwise it would cover residuals that other lanes still need.
    NERF_CHECK_ARG(y != residual || (d.out_dtype == d.dtype && (d.rows == 1u || d.y_stride == d.residual_stride)), "nerf_ext_linear_forward: y over residual must have its type and row stride");
    NERF_CHECK_ARG(aligned(workspace, 16u), "nerf_ext_linear_forward: workspace must be aligned to 16 bytes");
    const Workspace ws{(float*)workspace, workspace ? workspace_bytes : 0u};
    if (d.dtype == NERF_EXT_F16) return forward<half_t>(d, x, weight, bias, residual, y, pre, ws, (hipStream_t)stream);
    return forward<bf16_t>(d, x, weight, bias, residual, y, pre, ws, (hipStream_t)stream);
}

NERF_API NerfStatus nerf_ext_linear_backward(const NerfExtLinearDesc* desc, const void* x, const void* weight, const void* delta, const void* pre, const void* add, void* dx, void* dpre, float* dweight, float* dbias, void* workspace,
                                            uint64_t workspace_bytes, void* stream) {
    NerfExtLinearDesc d;
    const NerfStatus s = check_desc(desc, d, "nerf_ext_linear_backward");
    if (s != NERF_STATUS_OK) return s;
    NERF_CHECK_ARG(dx || dpre || dweight, "nerf_ext_linear_backward: no output");
    NERF_CHECK_ARG(!dbias || dweight, "nerf_ext_linear_backward: dbias comes with dweight only");
    NERF_CHECK_ARG(d.rows == 0u || delta, "nerf_ext_linear_backward: null delta");
    NERF_CHECK_ARG(d.rows == 0u || weight || !(dx || dpre), "nerf_ext_linear_backward: dx and dpre need weight");
    NERF_CHECK_ARG(d.rows == 0u || pre || !dpre, "nerf_ext_linear_backward: dpre needs pre");
    NERF_CHECK_ARG(d.rows == 0u || x || !dweight, "nerf_ext_linear_backward: dweight needs x");
    NERF_CHECK_ARG(aligned(x, 2u) && aligned(weight, 2u) && aligned(delta, 2u) && aligned(pre, 2u) && aligned(add, 2u) && aligned(dx, 2u) && aligned(dpre, 2u) && aligned(dweight, 4u) && aligned(dbias, 4u),
                   "nerf_ext_linear_backward: an array is not aligned to its elements");
    NERF_CHECK_ARG(aligned(workspace, 16u), "nerf_ext_linear_backward: workspace must be aligned to 16 bytes");
    if (d.rows == 0u && !dweight) return NERF_STATUS_OK;
    const Workspace ws{(float*)workspace, workspace ? workspace_bytes : 0u};
    if (d.dtype == NERF_EXT_F16) return backward<half_t>(d, x, weight, delta, pre, add, dx, dpre, dweight, dbias, ws, (hipStream_t)stream);
    return backward<bf16_t>(d, x, weight, delta, pre, add, dx, dpre, dweight, dbias, ws, (hipStream_t)stream);
}

}  // extern "C"
