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
// consecutive p of one q and stores them together.  An operand whose k is not
// contiguous is read from LDS through the transposing read
// (ds_read_b64_tr_b16), four k of one p a lane, so no operand is transposed in
// memory.  Products are of 16-bit values, exact in 32 bits, and summed in 32
// bits; y, pre, dx and dpre are rounded once, when they are stored.
#include <algorithm>

#include "common.hpp"

using namespace nerf_hip;

namespace {

typedef __bf16 bf16_t;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));

template <typename T>
struct Vec;
template <>
struct Vec<half_t> {
    using x4 = half4_t;
    using x8 = half8_t;
    static __device__ __forceinline__ floatx4 mfma(x8 a, x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Vec<bf16_t> {
    using x4 = bf16x4_t;
    using x8 = bf16x8_t;
    static __device__ __forceinline__ floatx4 mfma(x8 a, x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// ------------------------------------------------------------ activations
// sigma(t) = 1 / (1 + e^-t) and sigma'(t) = e^-|t| / (1 + e^-|t|)^2, which
// keeps its relative accuracy in both tails.
__device__ __forceinline__ float sigmoid(float t) { return __builtin_amdgcn_rcpf(1.0f + __expf(-t)); }
__device__ __forceinline__ float sigmoid_slope(float t) {
    const float e = __expf(-fabsf(t));
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    return e * r * r;
}

constexpr float kGeluA = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

template <uint32_t kAct>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (kAct == NERF_EXT_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
    if constexpr (kAct == NERF_EXT_ACT_SOFTPLUS) {
        // max(z, 0) + log(1 + e), e = exp(-|z|); log(1 + e) as e log(u) / (u - 1)
        // with u = 1 + e rounded, which is accurate for small e (Goldberg, "What
        // every computer scientist should know about floating-point
        // arithmetic", 1991, theorem 4).
        const float e = __expf(-fabsf(z));
        const float u = 1.0f + e, d = u - 1.0f;
        const float l = d == 0.0f ? e : e * __logf(u) * __builtin_amdgcn_rcpf(d);
        return (z < 0.0f ? 0.0f : z) + l;
    }
    if constexpr (kAct == NERF_EXT_ACT_SIGMOID) return sigmoid(z);
    if constexpr (kAct == NERF_EXT_ACT_SILU) return z * sigmoid(z);
    if constexpr (kAct == NERF_EXT_ACT_GELU) return z * sigmoid(2.0f * kGeluA * z * (1.0f + kGeluB * z * z));  // (1 + tanh u) / 2 = sigma(2u)
    return z;
}

template <uint32_t kAct>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (kAct == NERF_EXT_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (kAct == NERF_EXT_ACT_SOFTPLUS) return sigmoid(z);
    if constexpr (kAct == NERF_EXT_ACT_SIGMOID) return sigmoid_slope(z);
    if constexpr (kAct == NERF_EXT_ACT_SILU) return sigmoid(z) + z * sigmoid_slope(z);
    if constexpr (kAct == NERF_EXT_ACT_GELU) {
        // The second term vanishes beyond |z| = 16: clamped, its factors stay finite.
        const float c = fminf(fmaxf(z, -16.0f), 16.0f), t = 2.0f * kGeluA * c * (1.0f + kGeluB * c * c);
        return sigmoid(t) + c * sigmoid_slope(t) * (2.0f * kGeluA) * (1.0f + 3.0f * kGeluB * c * c);
    }
    return 1.0f;
}

// f(constant of the activation): one branch for a whole tile.
template <typename F>
__device__ __forceinline__ void with_activation(uint32_t act, F&& f) {
    switch (act) {
    case NERF_EXT_ACT_RELU: f(std::integral_constant<uint32_t, NERF_EXT_ACT_RELU>{}); break;
    case NERF_EXT_ACT_SOFTPLUS: f(std::integral_constant<uint32_t, NERF_EXT_ACT_SOFTPLUS>{}); break;
    case NERF_EXT_ACT_SIGMOID: f(std::integral_constant<uint32_t, NERF_EXT_ACT_SIGMOID>{}); break;
    case NERF_EXT_ACT_SILU: f(std::integral_constant<uint32_t, NERF_EXT_ACT_SILU>{}); break;
    case NERF_EXT_ACT_GELU: f(std::integral_constant<uint32_t, NERF_EXT_ACT_GELU>{}); break;
    default: f(std::integral_constant<uint32_t, NERF_EXT_ACT_NONE>{}); break;
    }
}

// ------------------------------------------------------------- epilogues
// What becomes of a finished sum.  Each gets four consecutive p of one q at a
// time, q < nq, p < np; vec: all four exist and every array's four are one
// aligned access.
template <typename T>
__device__ __forceinline__ floatx4 load4(const T* p, uint32_t n, bool vec) {
    if (vec) {
        const typename Vec<T>::x4 v = *reinterpret_cast<const typename Vec<T>::x4*>(p);
        return floatx4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    }
    floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t r = 0; r < 4u; ++r)
        if (r < n) o[r] = (float)p[r];
    return o;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, floatx4 v, uint32_t n, bool vec) {
    if (vec) {
        typename Vec<T>::x4 h;
#pragma unroll
        for (int r = 0; r < 4; ++r) h[r] = (T)v[r];
        *reinterpret_cast<typename Vec<T>::x4*>(p) = h;
        return;
    }
#pragma unroll
    for (uint32_t r = 0; r < 4u; ++r)
        if (r < n) p[r] = (T)v[r];
}
__device__ __forceinline__ void store4(float* p, floatx4 v, uint32_t n, bool vec) {
    if (vec) {
        *reinterpret_cast<floatx4*>(p) = v;
        return;
    }
#pragma unroll
    for (uint32_t r = 0; r < 4u; ++r)
        if (r < n) p[r] = v[r];
}

template <typename T>
struct ForwardOut {
    const float* bias;
    const T* residual;
    void* y;
    T* pre;
    uint64_t ldr, ldy;
    uint32_t np, nq, act;
    bool y32, vec;

    template <uint32_t kAct>
    __device__ __forceinline__ void put(uint32_t q, uint32_t p, floatx4 z) const {
        const uint32_t n = np - p;
        if (bias) {
#pragma unroll
            for (uint32_t r = 0; r < 4u; ++r)
                if (vec || r < n) z[r] += bias[p + r];
        }
        if (pre) store4(pre + (uint64_t)q * np + p, z, n, vec);
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = act_value<kAct>(z[r]);
        if (residual) {
            const floatx4 a = load4(residual + (uint64_t)q * ldr + p, n, vec);
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] += a[r];
        }
        if (y32) store4((float*)y + (uint64_t)q * ldy + p, z, n, vec);
        else store4((T*)y + (uint64_t)q * ldy + p, z, n, vec);
    }
};

template <typename T>
struct InputGradientOut {
    const T* add;
    T* dx;
    const T* pre;
    T* dpre;
    uint64_t ldx;
    uint32_t np, nq, act;
    bool vec;

    template <uint32_t kAct>
    __device__ __forceinline__ void put(uint32_t q, uint32_t p, floatx4 g) const {
        const uint32_t n = np - p;
        if (add) {
            const floatx4 a = load4(add + (uint64_t)q * ldx + p, n, vec);
#pragma unroll
            for (int r = 0; r < 4; ++r) g[r] += a[r];
        }
        if (dx) store4(dx + (uint64_t)q * ldx + p, g, n, vec);
        if (dpre) {
            const floatx4 z = load4(pre + (uint64_t)q * np + p, n, vec);
#pragma unroll
            for (int r = 0; r < 4; ++r) g[r] *= act_slope<kAct>(z[r]);
            store4(dpre + (uint64_t)q * np + p, g, n, vec);
        }
    }
};

// Plain sums in 32 bits: dW, or one part of a sum that was split over k.
struct SumOut {
    float* out;
    uint64_t part;  // elements from one part to the next
    float* row_sums;  // sum_k Q(q, k), or null; nq of them a part
    uint32_t np, nq, act;
    bool vec;
    template <uint32_t kAct>
    __device__ __forceinline__ void put(uint32_t q, uint32_t p, floatx4 v) const { store4(out + (uint64_t)q * np + p, v, np - p, vec); }
};

// ----------------------------------------------------------------- product
constexpr uint32_t kBK = 64u;  // k per tile: two matrix instructions' worth
constexpr uint32_t kThreads = 256u;

struct Operands {
    const void* p;
    const void* q;
    uint64_t ldp, ldq;  // elements between rows in memory
    uint32_t np, nq, nk;
    uint32_t k_split;   // k per part, a multiple of kBK
};

// A tile of kB rows x 64 k lies in LDS in 16-byte chunks of 8 values, the
// chunk's place xor-ed with bits of its row so that the lanes of one read
// fall on different banks: k contiguous, row-major [kB][64], the 8 rows of a
// read's lanes in 8 different places; kT (row contiguous), k-major [64][kB],
// the four k of a transposing read 32 bytes apart.
template <uint32_t kB, bool kT>
__device__ __forceinline__ uint32_t chunk_slot(uint32_t row, uint32_t chunk) {
    if constexpr (kT) return row * (kB / 8u) + (chunk ^ ((row & 3u) << 1));
    else return row * 8u + (chunk ^ (row & 7u));
}

// Tile [row0, row0 + kB) x [k0, k0 + 64) into LDS, zeros outside [0, n) x [0, nk).
template <typename T, uint32_t kB, bool kT>
__device__ __forceinline__ void stage(const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end, uint4* lds) {
    constexpr uint32_t kChunks = kT ? kB / 8u : 8u;
#pragma unroll
    for (uint32_t s = threadIdx.x; s < kB * 8u; s += kThreads) {
        const uint32_t line = s / kChunks;
        const uint32_t chunk = s % kChunks;
        const uint32_t major = (kT ? k0 : row0) + line, minor = (kT ? row0 : k0) + 8u * chunk;
        const uint32_t major_end = kT ? k_end : n, minor_end = kT ? n : k_end;
        uint4 v = {0u, 0u, 0u, 0u};
        if (major < major_end && minor < minor_end) {
            const T* at = src + (uint64_t)major * ld + minor;
            if (minor + 8u <= minor_end) {
                __builtin_memcpy(&v, at, 16);
            } else {
                short8_t h = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (uint32_t j = 0; j < 7u; ++j)
                    if (minor + j < minor_end) h[j] = __builtin_bit_cast(short, at[j]);
                v = __builtin_bit_cast(uint4, h);
            }
        }
        lds[chunk_slot<kB, kT>(line, chunk)] = v;
    }
}

// The 8 k of rows [row0, row0 + 16) that a lane feeds to one 16x16x32 matrix
// instruction: k = 32 step + 8 (lane / 16) + 0..7 of row row0 + lane % 16.
template <typename T, uint32_t kB, bool kT>
__device__ __forceinline__ typename Vec<T>::x8 fragment(const uint4* lds, uint32_t row0, uint32_t step) {
    const uint32_t lane = threadIdx.x & 63u, i = lane & 15u, g = lane >> 4;
    if constexpr (!kT) {
        return __builtin_bit_cast(typename Vec<T>::x8, lds[chunk_slot<kB, false>(row0 + i, 4u * step + g)]);
    } else {
        // Lane 4 r + c of 16 reads rows row0 + 4 c .. + 3 at k = r; the read hands
        // lane i the four k of row row0 + i.
        short4_t h[2];
#pragma unroll
        for (uint32_t half = 0; half < 2u; ++half) {
            const uint32_t k = 32u * step + 8u * g + 4u * half + (i >> 2), row = row0 + 4u * (i & 3u);
            const char* at = reinterpret_cast<const char*>(lds) + 16u * chunk_slot<kB, true>(k, row >> 3) + 2u * (row & 7u);
            h[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(at));
        }
        return __builtin_bit_cast(typename Vec<T>::x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, bool kPT, bool kQT, typename Out>
__global__ __launch_bounds__(kThreads) void k_product(Operands A, Out out) {
    static_assert(kWP * kWQ * 64u == kThreads);
    constexpr uint32_t kFP = kBP / kWP / 16u, kFQ = kBQ / kWQ / 16u;
    __shared__ uint4 lds_p[kBP * 8u];
    __shared__ uint4 lds_q[kBQ * 8u];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wp = (wave % kWP) * (kBP / kWP), wq = (wave / kWP) * (kBQ / kWQ);
    const uint32_t p0 = blockIdx.x * kBP, q0 = blockIdx.y * kBQ;
    const uint32_t k0 = blockIdx.z * A.k_split, k_end = min(A.nk, k0 + A.k_split);

    floatx4 acc[kFP][kFQ], sums[kFQ];
#pragma unroll
    for (uint32_t j = 0; j < kFQ; ++j) {
        sums[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t i = 0; i < kFP; ++i) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bool take_sums = false;
    if constexpr (std::is_same_v<Out, SumOut>) take_sums = out.row_sums && blockIdx.x == 0u && wp == 0u;
    typename Vec<T>::x8 ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = (T)1.0f;

    for (uint32_t k = k0; k < k_end; k += kBK) {
        stage<T, kBP, kPT>((const T*)A.p, A.ldp, A.np, p0, k, k_end, lds_p);
        stage<T, kBQ, kQT>((const T*)A.q, A.ldq, A.nq, q0, k, k_end, lds_q);
        __syncthreads();
#pragma unroll
        for (uint32_t step = 0; step < 2u; ++step) {
            typename Vec<T>::x8 fp[kFP], fq[kFQ];
#pragma unroll
            for (uint32_t i = 0; i < kFP; ++i) fp[i] = fragment<T, kBP, kPT>(lds_p, wp + 16u * i, step);
#pragma unroll
            for (uint32_t j = 0; j < kFQ; ++j) fq[j] = fragment<T, kBQ, kQT>(lds_q, wq + 16u * j, step);
#pragma unroll
            for (uint32_t i = 0; i < kFP; ++i)
#pragma unroll
                for (uint32_t j = 0; j < kFQ; ++j) acc[i][j] = Vec<T>::mfma(fp[i], fq[j], acc[i][j]);
            if constexpr (std::is_same_v<Out, SumOut>) {
                if (take_sums) {
#pragma unroll
                    for (uint32_t j = 0; j < kFQ; ++j) sums[j] = Vec<T>::mfma(ones, fq[j], sums[j]);
                }
            }
        }
        __syncthreads();
    }

    if constexpr (std::is_same_v<Out, SumOut>) {
        out.out += blockIdx.z * out.part;
        if (take_sums && lane < 16u) {  // every p of the product with ones holds the sum
#pragma unroll
            for (uint32_t j = 0; j < kFQ; ++j) {
                const uint32_t q = q0 + wq + 16u * j + lane;
                if (q < out.nq) out.row_sums[(uint64_t)blockIdx.z * out.nq + q] = sums[j][0];
            }
        }
    }
    with_activation(out.act, [&](auto act) {
#pragma unroll
        for (uint32_t j = 0; j < kFQ; ++j) {
            const uint32_t q = q0 + wq + 16u * j + (lane & 15u);
#pragma unroll
            for (uint32_t i = 0; i < kFP; ++i) {
                const uint32_t p = p0 + wp + 16u * i + 4u * (lane >> 4);
                if (q < out.nq && p < out.np) out.template put<act()>(q, p, acc[i][j]);
            }
        }
    });
}

// Joins the parts of a sum that was split over k, in their order.
template <typename Out>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ parts, uint64_t part, uint32_t count, const float* __restrict__ sums, float* __restrict__ row_sums, Out out) {
    const uint32_t quads = (out.np + 3u) / 4u;
    const uint64_t total = (uint64_t)quads * out.nq, step = (uint64_t)gridDim.x * blockDim.x, first = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    with_activation(out.act, [&](auto act) {
        for (uint64_t at = first; at < total; at += step) {
            const uint32_t q = (uint32_t)(at / quads), p = 4u * (uint32_t)(at % quads);
            floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t c = 0; c < count; ++c) {
                const float* src = parts + c * part + (uint64_t)q * out.np + p;
                if (out.vec) {
                    v += *reinterpret_cast<const floatx4*>(src);
                } else {
#pragma unroll
                    for (uint32_t r = 0; r < 4u; ++r)
                        if (p + r < out.np) v[r] += src[r];
                }
            }
            out.template put<act()>(q, p, v);
        }
    });
    if (row_sums) {
        for (uint64_t q = first; q < out.nq; q += step) {
            float s = 0.0f;
            for (uint32_t c = 0; c < count; ++c) s += sums[(uint64_t)c * out.nq + q];
            row_sums[q] = s;
        }
    }
}

// ------------------------------------------------------------------- host
constexpr uint32_t kMaxFeatures = 1u << 16, kMaxStride = 1u << 22, kMaxRows = 1u << 30;

bool aligned(const void* p, uint64_t bytes) { return ((uintptr_t)p & (bytes - 1u)) == 0u; }
uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1u) / b); }

struct Workspace {
    float* data;
    uint64_t bytes;
};

template <typename T, bool kPT, bool kQT, typename Out>
hipError_t launch_product(Operands A, Out out, float* row_sums, Workspace ws, hipStream_t stream) {
    constexpr uint32_t kBP = 64u, kBQ = 64u;
    const uint32_t tp = ceil_div(A.np, kBP), tq = ceil_div(A.nq, kBQ);
    // Split over k until every CU has two workgroups, with four tiles of k a
    // part at least, as far as the workspace holds the parts.
    const uint64_t part = (uint64_t)A.np * A.nq;
    const uint64_t per = 4u * (part + (row_sums ? A.nq : 0u));
    uint64_t splits = (2ull * device_cu_count()) / ((uint64_t)tp * tq);
    splits = std::min<uint64_t>({splits, ceil_div(A.nk, 4u * kBK), ws.data ? ws.bytes / per : 0u, 65535u});
    const bool split = splits > 1u;
    if (!split) splits = 1u;
    A.k_split = ceil_div(ceil_div(A.nk, kBK), splits) * kBK;
    if (A.k_split == 0u) A.k_split = kBK;
    const uint32_t parts = std::max(1u, ceil_div(A.nk, A.k_split));
    const dim3 grid(tp, tq, parts);
    if (parts > 1u) {
        float* sums = row_sums ? ws.data + parts * part : nullptr;
        const SumOut so{ws.data, part, sums, A.np, A.nq, NERF_EXT_ACT_NONE, A.np % 4u == 0u};
        k_product<T, kBP, kBQ, 2, 2, kPT, kQT, SumOut><<<grid, kThreads, 0, stream>>>(A, so);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        const uint64_t quads = (uint64_t)ceil_div(A.np, 4u) * A.nq;
        k_join<Out><<<(uint32_t)std::min<uint64_t>(ceil_div(quads, 256u), 4096u), 256, 0, stream>>>(ws.data, part, parts, sums, row_sums, out);
        return hipGetLastError();
    }
    k_product<T, kBP, kBQ, 2, 2, kPT, kQT, Out><<<grid, kThreads, 0, stream>>>(A, out);
    return hipGetLastError();
}

// rows beyond gridDim's range of 64-row tiles are taken in launches of this many.
constexpr uint32_t kRowsPerLaunch = 65535u * 64u;

template <typename T>
NerfStatus forward(const NerfExtLinearDesc& d, const void* x, const void* w, const float* bias, const void* residual, void* y, void* pre, Workspace ws, hipStream_t stream) {
    const bool y32 = d.out_dtype == NERF_EXT_F32;
    const bool vec = d.out_features % 4u == 0u && d.y_stride % 4u == 0u && aligned(y, y32 ? 16u : 8u) && aligned(bias, 16u) && (!pre || aligned(pre, 8u)) && (!residual || (d.residual_stride % 4u == 0u && aligned(residual, 8u)));
    for (uint64_t r0 = 0; r0 < d.rows; r0 += kRowsPerLaunch) {
        const uint32_t n = (uint32_t)std::min<uint64_t>(kRowsPerLaunch, d.rows - r0);
        const Operands A{w, (const T*)x + r0 * d.x_stride, d.in_features, d.x_stride, d.out_features, n, d.in_features, 0u};
        void* yo = y32 ? (void*)((float*)y + r0 * d.y_stride) : (void*)((T*)y + r0 * d.y_stride);
        const ForwardOut<T> out{bias, residual ? (const T*)residual + r0 * d.residual_stride : nullptr, yo, pre ? (T*)pre + r0 * d.out_features : nullptr, d.residual_stride, d.y_stride, d.out_features, n, d.activation, y32, vec};
        NERF_HIP_TRY((launch_product<T, false, false>(A, out, nullptr, ws, stream)));
    }
    return NERF_STATUS_OK;
}

template <typename T>
NerfStatus backward(const NerfExtLinearDesc& d, const void* x, const void* w, const void* delta, const void* pre, const void* add, void* dx, void* dpre, float* dw, float* db, Workspace ws, hipStream_t stream) {
    if (dx || dpre) {
        const bool vec = d.in_features % 4u == 0u && (!(add || dx) || d.x_stride % 4u == 0u) && aligned(add, 8u) && aligned(dx, 8u) && aligned(pre, 8u) && aligned(dpre, 8u);
        for (uint64_t r0 = 0; r0 < d.rows; r0 += kRowsPerLaunch) {
            const uint32_t n = (uint32_t)std::min<uint64_t>(kRowsPerLaunch, d.rows - r0);
            const Operands A{w, (const T*)delta + r0 * d.y_stride, d.in_features, d.y_stride, d.in_features, n, d.out_features, 0u};
            const InputGradientOut<T> out{add ? (const T*)add + r0 * d.x_stride : nullptr, dx ? (T*)dx + r0 * d.x_stride : nullptr, pre ? (const T*)pre + r0 * d.in_features : nullptr,
                                          dpre ? (T*)dpre + r0 * d.in_features : nullptr, d.x_stride, d.in_features, n, d.activation, vec};
            NERF_HIP_TRY((launch_product<T, true, false>(A, out, nullptr, ws, stream)));
        }
    }
    if (dw) {
        const Operands A{x, delta, d.x_stride, d.y_stride, d.in_features, d.out_features, d.rows, 0u};
        const SumOut out{dw, 0u, db, d.in_features, d.out_features, NERF_EXT_ACT_NONE, d.in_features % 4u == 0u && aligned(dw, 16u)};
        NERF_HIP_TRY((launch_product<T, true, true>(A, out, db, ws, stream)));
    }
    return NERF_STATUS_OK;
}

NerfStatus check_desc(const NerfExtLinearDesc* desc, NerfExtLinearDesc& d, const char* fn) {
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
    if (d.x_stride > kMaxStride || d.y_stride > kMaxStride || d.residual_stride > kMaxStride) return refuse("a row stride is above 2^22");
    return NERF_STATUS_OK;
}

}  // namespace

extern "C" {

NERF_API NerfStatus nerf_ext_linear_forward(const NerfExtLinearDesc* desc, const void* x, const void* weight, const float* bias, const void* residual, void* y, void* pre, void* workspace, uint64_t workspace_bytes, void* stream) {
    NerfExtLinearDesc d;
    const NerfStatus s = check_desc(desc, d, "nerf_ext_linear_forward");
    if (s != NERF_STATUS_OK) return s;
    if (d.rows == 0u) return NERF_STATUS_OK;
    NERF_CHECK_ARG(x && weight && y, "nerf_ext_linear_forward: null x, weight or y");
    NERF_CHECK_ARG(aligned(x, 2u) && aligned(weight, 2u) && aligned(residual, 2u) && aligned(pre, 2u) && aligned(bias, 4u) && aligned(y, d.out_dtype == NERF_EXT_F32 ? 4u : 2u), "nerf_ext_linear_forward: an array is not aligned to its elements");
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
    const Workspace ws{(float*)workspace, workspace ? workspace_bytes : 0u};
    if (d.dtype == NERF_EXT_F16) return backward<half_t>(d, x, weight, delta, pre, add, dx, dpre, dweight, dbias, ws, (hipStream_t)stream);
    return backward<bf16_t>(d, x, weight, delta, pre, add, dx, dpre, dweight, dbias, ws, (hipStream_t)stream);
}

}  // extern "C"
