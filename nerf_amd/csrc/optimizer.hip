// optimizer.hip — the norm and clipping of gradients that lie in many tensors,
// and the trainer's Adam update on a caller's tensors (include/nerf_ext.h,
// nerf_ext_grad_norm, nerf_ext_grad_clip, nerf_ext_adam_step).
//
// A launch covers many tensors: their pointers and lengths travel as kernel
// arguments, and a workgroup finds the tensor of its piece by the pieces'
// running count.  Squares are summed in 64 bits, per workgroup and then over
// the workgroups in their order, so that the norm is the same every time and
// neither overflows nor loses small gradients beside large ones.
#include <math.h>

#include <algorithm>

#include "common.hpp"

using namespace nerf_hip;

namespace {

typedef __bf16 bf16_t;

constexpr uint32_t kThreads  = 256u;
constexpr uint32_t kPiece    = 2048u;  // elements of a workgroup's turn
constexpr uint32_t kMaxParts = NERF_EXT_NORM_WORKSPACE / sizeof(double);

// Kernel arguments are kept below 4 KiB.
constexpr uint32_t kNormListed = 128u, kAdamListed = 64u;
struct NormList {
    const void* data[kNormListed];
    void* out[kNormListed];
    uint32_t first[kNormListed + 1u];  // pieces before the tensor's; all pieces behind the last
    uint16_t tail[kNormListed];        // elements of its last piece
    uint8_t dtype[kNormListed];
    uint32_t tensors, pieces, workers;
};
struct AdamList {
    float* param[kAdamListed];
    const float* grad[kAdamListed];
    float* m[kAdamListed];
    float* v[kAdamListed];
    void* copy[kAdamListed];
    uint32_t first[kAdamListed + 1u];
    uint16_t tail[kAdamListed];
    uint8_t dtype[kAdamListed];
    uint32_t tensors, pieces, workers;
};

// Worker w (a workgroup, or a wave of one) has every l.workers-th piece from w on
// or (kBack) the same from the list's end: a pass after another over the same
// tensors begins with what the one before read last, which the memory-side cache
// (256 MiB) still holds.  f(tensor, first element, elements).  Counts are 32-bit
// words: of a select between 64-bit lengths (the piece's end or the tensor's)
// the compiler kept the wrong condition here and let workgroups run past a
// tensor's end.
template <bool kBack, typename List, typename F>
__device__ __forceinline__ void each_piece(const List& l, uint32_t worker, F&& f) {
    if (worker >= l.pieces) return;
    // The tensor of the first piece to come: one less than those that start at
    // or before it, each lane asking for its own (a search by halves waited for
    // one load after another).
    uint32_t piece = kBack ? l.pieces - 1u - worker : worker, t = 0u;
    for (uint32_t base = 0; base < l.tensors; base += 64u) {
        const uint32_t i = base + (threadIdx.x & 63u);
        t += (uint32_t)__popcll(__ballot(i < l.tensors && l.first[i] <= piece));
    }
    t = __builtin_amdgcn_readfirstlane(t - 1u);
    for (uint32_t left = (l.pieces - 1u - worker) / l.workers + 1u; left > 0u; --left) {
        if (kBack) {
            while (piece < l.first[t]) --t;
        } else {
            while (piece >= l.first[t + 1u]) ++t;
        }
        f(t, (uint64_t)(piece - l.first[t]) * kPiece, piece + 1u == l.first[t + 1u] ? l.tail[t] : kPiece);
        piece = kBack ? piece - l.workers : piece + l.workers;
    }
}

// A lane's turn: 16 consecutive bytes, as 32-bit values, and back with one
// rounding; a wave's turn is one contiguous piece of memory (with 32 bytes a
// lane, fetched by two instructions, Adam ran at 5.0 TB/s, with 16 at 5.6).
// Arrays are aligned to their elements; the hardware serves wide accesses at
// any such address.
template <typename E, uint32_t kN>
struct Turn {
    typedef float Wide __attribute__((ext_vector_type(kN)));
    typedef E Narrow __attribute__((ext_vector_type(kN)));
    static __device__ __forceinline__ Wide load(const E* p) {
        Narrow v;
        __builtin_memcpy(&v, p, sizeof(v));
        return __builtin_convertvector(v, Wide);
    }
    static __device__ __forceinline__ void store(E* p, const Wide& v) {
        const Narrow h = __builtin_convertvector(v, Narrow);
        __builtin_memcpy(p, &h, sizeof(h));
    }
};

// f(pointer type tag) for an element type.
template <typename F>
__device__ __forceinline__ void with_type(uint32_t dtype, F&& f) {
    if (dtype == NERF_EXT_F32) f((float*)nullptr);
    else if (dtype == NERF_EXT_F16) f((half_t*)nullptr);
    else f((bf16_t*)nullptr);
}

// Sum over the workgroup, in thread 0.
template <uint32_t kCount>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double ws[kCount / 64u];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_down(v, d);
    if ((threadIdx.x & 63u) == 0u) ws[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (uint32_t w = 0; w < kCount / 64u; ++w) s += ws[w];
    return s;
}

// The sum of the squares of a worker's pieces, the share of it that lane `lane`
// of the worker's kLanes has.
template <uint32_t kLanes>
__device__ __forceinline__ double worker_squares(const NormList& l, uint32_t worker, uint32_t lane) {
    double s = 0.0;
    each_piece<false>(l, worker, [&](uint32_t t, uint64_t first, uint32_t n) {
        with_type(l.dtype[t], [&](auto* tag) {
            using E       = std::remove_pointer_t<decltype(tag)>;
            const E* data = (const E*)l.data[t] + first;
            constexpr uint32_t kN = 16u / sizeof(E), kTurns = kPiece / (kN * kLanes);
            if (n == kPiece) {
                typename Turn<E, kN>::Wide g[kTurns];
#pragma unroll
                for (uint32_t k = 0; k < kTurns; ++k) g[k] = Turn<E, kN>::load(data + kN * (k * kLanes + lane));
#pragma unroll
                for (uint32_t k = 0; k < kTurns; ++k)
#pragma unroll
                    for (uint32_t r = 0; r < kN; ++r) s += (double)g[k][r] * (double)g[k][r];
            } else {
                for (uint32_t i = lane; i < n; i += kLanes) {
                    const double g = (double)(float)data[i];
                    s += g * g;
                }
            }
        });
    });
    return s;
}

// parts[b] = sum of the squares of workgroup b's pieces.  Bound by memory; pieces
// in turn over the workgroups read and clip 48 gradients of 2048 x 2048 in 466 us, a
// contiguous share each in 483.
__global__ __launch_bounds__(kThreads) void k_square_sums(NormList l, double* __restrict__ parts) {
    const double s = block_sum<kThreads>(worker_squares<kThreads>(l, blockIdx.x, threadIdx.x));
    if (threadIdx.x == 0u) parts[blockIdx.x] = s;
}

// A short list's norm in one launch: one workgroup, whose waves share the pieces.
// Bound by the launch: 6 us for up to 64 pieces, two launches 9.
constexpr uint32_t kShortThreads = 1024u, kShortWaves = kShortThreads / 64u;
constexpr uint32_t kShortPieces  = 4u * kShortWaves;
__global__ __launch_bounds__(kShortThreads) void k_norm_short(NormList l, float* __restrict__ norm) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const double s      = block_sum<kShortThreads>(worker_squares<64u>(l, wave, threadIdx.x & 63u));
    if (threadIdx.x == 0u) *norm = (float)sqrt(s);
}

// sqrt of the sum of all parts, the same in every workgroup and thread.
__device__ __forceinline__ float norm_of(const double* __restrict__ parts, uint32_t n) {
    __shared__ double total;
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) s += parts[i];
    s = block_sum<kThreads>(s);
    if (threadIdx.x == 0u) total = s;
    __syncthreads();
    return (float)sqrt(total);
}

__global__ __launch_bounds__(kThreads) void k_norm(const double* __restrict__ parts, uint32_t n, float* __restrict__ norm) {
    const float v = norm_of(parts, n);
    if (threadIdx.x == 0u) *norm = v;
}

// out = grad * min(1, max_norm / norm); each workgroup adds up the parts itself,
// which saves a launch.  Bound by memory: one read and one write, after the
// norm's read, part of which the memory-side cache still holds.
__global__ __launch_bounds__(kThreads) void k_clip(NormList l, const double* __restrict__ parts, uint32_t n, float max_norm, float* __restrict__ norm) {
    const float v      = norm_of(parts, n);
    const float factor = v > max_norm && isfinite(v) ? max_norm / v : 1.0f;
    if (blockIdx.x == 0u && threadIdx.x == 0u) *norm = v;
    each_piece<true>(l, blockIdx.x, [&](uint32_t t, uint64_t first, uint32_t n) {
        with_type(l.dtype[t], [&](auto* tag) {
            using E       = std::remove_pointer_t<decltype(tag)>;
            const E* data = (const E*)l.data[t] + first;
            E* out        = (E*)l.out[t] + first;
            constexpr uint32_t kN = 16u / sizeof(E), kTurns = kPiece / (kN * kThreads);
            if (n == kPiece) {
                typename Turn<E, kN>::Wide g[kTurns];
#pragma unroll
                for (uint32_t k = 0; k < kTurns; ++k) g[k] = Turn<E, kN>::load(data + kN * (k * kThreads + threadIdx.x));
#pragma unroll
                for (uint32_t k = 0; k < kTurns; ++k) Turn<E, kN>::store(out + kN * (k * kThreads + threadIdx.x), g[k] * factor);
            } else {
                for (uint32_t i = threadIdx.x; i < n; i += kThreads) out[i] = (E)((float)data[i] * factor);
            }
        });
    });
}

struct AdamRule {
    float lr, beta1, beta2, eps, bc1, bc2, clip, guard, loss_scale;
};

//   m = b1 m + (1 - b1) g   v = b2 v + (1 - b2) g^2   p -= lr (m bc1) / (sqrt(v bc2) + eps)
// with g the gradient over the loss scale, clipped.  Bound by memory: 28 bytes a
// parameter, 30 with a 16-bit copy, at 4.8 to 5.3 TB/s (a copy's rate is 5.1).
__global__ __launch_bounds__(kThreads) void k_adam_tensors(AdamList l, AdamRule r, const float* __restrict__ norm, uint32_t* __restrict__ skipped) {
    const float gn  = *norm / r.loss_scale;
    const bool skip = !isfinite(gn) || gn > r.guard;
    if (skipped && blockIdx.x == 0u && threadIdx.x == 0u) *skipped = skip ? 1u : 0u;
    if (skip) return;
    const float gs = (gn > r.clip && gn > 0.0f ? r.clip / gn : 1.0f) * (1.0f / r.loss_scale);
    each_piece<true>(l, blockIdx.x, [&](uint32_t t, uint64_t first, uint32_t n) {
        float *param = l.param[t] + first, *ms = l.m[t] + first, *vs = l.v[t] + first;
        const float* grad = l.grad[t] + first;
        void* copy        = l.copy[t];
        const auto one = [&](float& p, float g, float& m, float& v) {
            g *= gs;
            m = r.beta1 * m + (1.0f - r.beta1) * g;
            v = r.beta2 * v + (1.0f - r.beta2) * g * g;
            p = p - r.lr * (m * r.bc1) / (sqrtf(v * r.bc2) + r.eps);
        };
        if (n == kPiece) {
            using F4 = Turn<float, 4u>;
            // The next turn's values are on their way while this one's are written.
            F4::Wide p[2], m[2], v[2], g[2];
            auto fetch = [&](uint32_t k) {
                const uint32_t i = 4u * (k * kThreads + threadIdx.x);
                p[k & 1u] = F4::load(param + i);
                m[k & 1u] = F4::load(ms + i);
                v[k & 1u] = F4::load(vs + i);
                g[k & 1u] = F4::load(grad + i);
            };
            constexpr uint32_t kTurns = kPiece / (4u * kThreads);
            fetch(0u);
#pragma unroll
            for (uint32_t k = 0; k < kTurns; ++k) {
                const uint32_t i = 4u * (k * kThreads + threadIdx.x), h = k & 1u;
                if (k + 1u < kTurns) fetch(k + 1u);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float pe = p[h][e], me = m[h][e], ve = v[h][e];
                    one(pe, g[h][e], me, ve);
                    p[h][e] = pe;
                    m[h][e] = me;
                    v[h][e] = ve;
                }
                F4::store(param + i, p[h]);
                F4::store(ms + i, m[h]);
                F4::store(vs + i, v[h]);
                if (copy && l.dtype[t] == NERF_EXT_F16) Turn<half_t, 4u>::store((half_t*)copy + first + i, p[h]);
                else if (copy) Turn<bf16_t, 4u>::store((bf16_t*)copy + first + i, p[h]);
            }
        } else {
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
                float p = param[i], m = ms[i], v = vs[i];
                one(p, grad[i], m, v);
                param[i] = p;
                ms[i]    = m;
                vs[i]    = v;
                if (copy && l.dtype[t] == NERF_EXT_F16) ((half_t*)copy)[first + i] = (half_t)p;
                else if (copy) ((bf16_t*)copy)[first + i] = (bf16_t)p;
            }
        }
    });
}

// ------------------------------------------------------------------- host
uint64_t element_bytes(uint32_t dtype) { return dtype == NERF_EXT_F32 ? 4u : 2u; }
bool aligned(const void* p, uint64_t bytes) { return (uintptr_t)p % bytes == 0u; }

NerfStatus refuse(const char* fn, const char* why) {
    set_error(std::string(fn) + ": " + why);
    return NERF_STATUS_INVALID_USAGE;
}

// Pieces of a list (128 tensors at most) fit 32 bits: 2^23 each.
constexpr uint64_t kMaxCount   = (uint64_t)kPiece << 23;
constexpr uint32_t kMaxTensors = 1u << 20;                // a list has a part at least

NerfStatus check_grads(const char* fn, const NerfExtGradTensor* tensors, uint32_t count, const float* norm, const void* workspace, uint64_t bytes, bool outputs) {
    if (count && !tensors) return refuse(fn, "null tensor list");
    if (count > kMaxTensors) return refuse(fn, "more than 2^20 tensors");
    if (!norm || !aligned(norm, 4u)) return refuse(fn, "norm must be a device float");
    if (!workspace || bytes < NERF_EXT_NORM_WORKSPACE || !aligned(workspace, 16u)) return refuse(fn, "workspace must have NERF_EXT_NORM_WORKSPACE bytes, aligned to 16");
    for (uint32_t i = 0; i < count; ++i) {
        const NerfExtGradTensor& t = tensors[i];
        if (t.dtype != NERF_EXT_F32 && t.dtype != NERF_EXT_F16 && t.dtype != NERF_EXT_BF16) return refuse(fn, "unknown dtype of a tensor");
        if (t.reserved != 0u) return refuse(fn, "reserved must be 0");
        if (t.count > kMaxCount) return refuse(fn, "a tensor has more than 2^34 elements");
        if (t.count && (!t.grad || (outputs && !t.out))) return refuse(fn, "null data of a tensor");
        if (!aligned(t.grad, element_bytes(t.dtype)) || (outputs && !aligned(t.out, element_bytes(t.dtype)))) return refuse(fn, "a tensor is not aligned to its elements");
    }
    return NERF_STATUS_OK;
}

// f(list, workgroups) for the tensors, in lists of at most the arguments' size
// and with at most `most` workgroups a list; empty tensors are left out.
template <typename List, uint32_t kListed, typename Tensor, typename Put, typename F>
hipError_t each_list(const Tensor* tensors, uint32_t count, uint32_t most, Put&& put, F&& f) {
    for (uint32_t at = 0; at < count;) {
        List l;
        l.tensors = l.pieces = 0u;
        for (; at < count && l.tensors < kListed; ++at) {
            const uint64_t n = tensors[at].count;
            if (n == 0u) continue;
            l.first[l.tensors] = l.pieces;
            l.tail[l.tensors]  = (uint16_t)((n - 1u) % kPiece + 1u);
            put(l, l.tensors, tensors[at]);
            l.pieces += (uint32_t)((n + kPiece - 1u) / kPiece);
            ++l.tensors;
        }
        if (l.tensors == 0u) break;
        l.first[l.tensors] = l.pieces;
        l.workers          = std::min(l.pieces, most);
        const hipError_t e = f(l, l.workers);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

void put_grad(NormList& l, uint32_t i, const NerfExtGradTensor& t) {
    l.data[i]  = t.grad;
    l.out[i]   = t.out;
    l.dtype[i] = (uint8_t)t.dtype;
}

// The parts of all tensors' squares, *n of them.
hipError_t square_sums(const NerfExtGradTensor* tensors, uint32_t count, double* parts, uint32_t* n, hipStream_t stream) {
    const uint32_t lists = (count + kNormListed - 1u) / kNormListed;
    const uint32_t most  = std::max(1u, std::min(8u * device_cu_count(), kMaxParts / std::max(1u, lists)));
    *n = 0u;
    return each_list<NormList, kNormListed>(tensors, count, most, put_grad, [&](const NormList& l, uint32_t blocks) {
        k_square_sums<<<blocks, kThreads, 0, stream>>>(l, parts + *n);
        *n += blocks;
        return hipGetLastError();
    });
}

}  // namespace

extern "C" {

NERF_API NerfStatus nerf_ext_grad_norm(const NerfExtGradTensor* tensors, uint32_t count, float* norm, void* workspace, uint64_t workspace_bytes, void* stream) {
    const NerfStatus s = check_grads("nerf_ext_grad_norm", tensors, count, norm, workspace, workspace_bytes, false);
    if (s != NERF_STATUS_OK) return s;
    // Up to 2^17 elements one workgroup takes 6 us, and two launches 9.
    if (count <= kNormListed) {
        uint64_t pieces = 0u;
        for (uint32_t i = 0; i < count; ++i) pieces += (tensors[i].count + kPiece - 1u) / kPiece;
        if (pieces > 0u && pieces <= kShortPieces) {
            NERF_HIP_TRY((each_list<NormList, kNormListed>(tensors, count, kShortWaves, put_grad, [&](const NormList& l, uint32_t) {
                k_norm_short<<<1, kShortThreads, 0, (hipStream_t)stream>>>(l, norm);
                return hipGetLastError();
            })));
            return NERF_STATUS_OK;
        }
    }
    uint32_t n = 0u;
    NERF_HIP_TRY(square_sums(tensors, count, (double*)workspace, &n, (hipStream_t)stream));
    k_norm<<<1, kThreads, 0, (hipStream_t)stream>>>((const double*)workspace, n, norm);
    NERF_LAUNCH_CHECK("k_norm");
    return NERF_STATUS_OK;
}

NERF_API NerfStatus nerf_ext_grad_clip(const NerfExtGradTensor* tensors, uint32_t count, float max_norm, float* norm, void* workspace, uint64_t workspace_bytes, void* stream) {
    const NerfStatus s = check_grads("nerf_ext_grad_clip", tensors, count, norm, workspace, workspace_bytes, true);
    if (s != NERF_STATUS_OK) return s;
    NERF_CHECK_ARG(max_norm >= 0.0f, "nerf_ext_grad_clip: max_norm must not be negative or NaN");
    uint32_t n = 0u;
    NERF_HIP_TRY(square_sums(tensors, count, (double*)workspace, &n, (hipStream_t)stream));
    if (n == 0u) {
        k_norm<<<1, kThreads, 0, (hipStream_t)stream>>>((const double*)workspace, 0u, norm);
        NERF_LAUNCH_CHECK("k_norm");
        return NERF_STATUS_OK;
    }
    NERF_HIP_TRY((each_list<NormList, kNormListed>(tensors, count, 8u * device_cu_count(), put_grad, [&](const NormList& l, uint32_t blocks) {
        k_clip<<<blocks, kThreads, 0, (hipStream_t)stream>>>(l, (const double*)workspace, n, max_norm, norm);
        return hipGetLastError();
    })));
    return NERF_STATUS_OK;
}

NERF_API NerfStatus nerf_ext_adam_step(const NerfExtAdamTensor* tensors, uint32_t count, const NerfHyperParams* hyper, uint32_t step, const float* grad_norm, uint32_t* skipped, void* stream) {
    const char* fn = "nerf_ext_adam_step";
    if (count && !tensors) return refuse(fn, "null tensor list");
    if (count > kMaxTensors) return refuse(fn, "more than 2^20 tensors");
    if (!hyper || !grad_norm || !aligned(grad_norm, 4u) || !aligned(skipped, 4u)) return refuse(fn, "null or unaligned hyper-parameters, grad_norm or skipped");
    if (step == 0u) return refuse(fn, "steps count from 1");
    if (!(hyper->loss_scale > 0.0f)) return refuse(fn, "loss_scale must be positive");
    if (!(hyper->adam_beta1 >= 0.0f && hyper->adam_beta1 < 1.0f && hyper->adam_beta2 >= 0.0f && hyper->adam_beta2 < 1.0f)) return refuse(fn, "betas must be in [0, 1)");
    for (uint32_t i = 0; i < count; ++i) {
        const NerfExtAdamTensor& t = tensors[i];
        if (t.copy && t.copy_dtype != NERF_EXT_F16 && t.copy_dtype != NERF_EXT_BF16) return refuse(fn, "copy_dtype must be NERF_EXT_F16 or NERF_EXT_BF16");
        if (t.reserved != 0u) return refuse(fn, "reserved must be 0");
        if (t.count > kMaxCount) return refuse(fn, "a tensor has more than 2^34 elements");
        if (t.count && (!t.param || !t.grad || !t.m || !t.v)) return refuse(fn, "null data of a tensor");
        if (!aligned(t.param, 4u) || !aligned(t.grad, 4u) || !aligned(t.m, 4u) || !aligned(t.v, 4u) || !aligned(t.copy, 2u)) return refuse(fn, "a tensor is not aligned to its elements");
    }
    // The trainer's coefficients (backend-cuda.cu:1513-1536), those that do not
    // depend on the norm computed here and in 64 bits (the trainer's kernel takes
    // its powers in 32: the same rule, not the same bits).
    const double decay = (double)hyper->lr_decay_ksteps * 1000.0;
    AdamRule r;
    r.lr         = decay > 0.0 ? (float)(hyper->learning_rate * pow(0.1, step / decay)) : hyper->learning_rate;
    r.beta1      = hyper->adam_beta1;
    r.beta2      = hyper->adam_beta2;
    r.eps        = hyper->adam_eps;
    r.bc1        = (float)(1.0 / (1.0 - pow((double)hyper->adam_beta1, step)));
    r.bc2        = (float)(1.0 / (1.0 - pow((double)hyper->adam_beta2, step)));
    r.clip       = hyper->grad_clip_norm;
    r.guard      = hyper->update_guard_grad_norm;
    r.loss_scale = hyper->loss_scale;
    bool first = true;
    NERF_HIP_TRY((each_list<AdamList, kAdamListed>(
        tensors, count, 8u * device_cu_count(),
        [](AdamList& l, uint32_t i, const NerfExtAdamTensor& t) {
            l.param[i] = t.param;
            l.grad[i]  = t.grad;
            l.m[i]     = t.m;
            l.v[i]     = t.v;
            l.copy[i]  = t.copy;
            l.dtype[i] = (uint8_t)t.copy_dtype;
        },
        [&](const AdamList& l, uint32_t blocks) {
            k_adam_tensors<<<blocks, kThreads, 0, (hipStream_t)stream>>>(l, r, grad_norm, first ? skipped : nullptr);
            first = false;
            return hipGetLastError();
        })));
    if (first && skipped) {  // nothing to update: the flag alone
        k_adam_tensors<<<1, kThreads, 0, (hipStream_t)stream>>>(AdamList{}, r, grad_norm, skipped);
        NERF_LAUNCH_CHECK("k_adam_tensors");
    }
    return NERF_STATUS_OK;
}

}  // extern "C"
