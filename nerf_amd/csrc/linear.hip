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
// bits; y, pre, dx and dpre are rounded once, when they are stored.
#include <algorithm>

#include "common.hpp"

using namespace nerf_hip;

namespace {

typedef __bf16 bf16_t;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));

template <typename T>
struct Vec;
template <>
struct Vec<half_t> {
    using x8 = half8_t;
    static __device__ __forceinline__ floatx4 mfma(x8 a, x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Vec<bf16_t> {
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
    if constexpr (kAct == NERF_EXT_ACT_SILU) {
        // The second term vanishes beyond |z| = 110: clamped, it does so at an
        // infinity too, as a finite z is stored beyond the range of 16 bits.
        const float c = z < -128.0f ? -128.0f : z > 128.0f ? 128.0f : z;
        return sigmoid(z) + c * sigmoid_slope(c);
    }
    if constexpr (kAct == NERF_EXT_ACT_GELU) {
        // The second term vanishes beyond |z| = 16: clamped, its factors stay finite,
        // and a NaN stays one.
        const float c = z < -16.0f ? -16.0f : z > 16.0f ? 16.0f : z, t = 2.0f * kGeluA * c * (1.0f + kGeluB * c * c);
        return sigmoid(t) + c * sigmoid_slope(t) * (2.0f * kGeluA) * (1.0f + 3.0f * kGeluB * c * c);
    }
    return 1.0f;
}

// act_value / act_slope of eight values, one branch for all of them.
typedef float floatx8 __attribute__((ext_vector_type(8)));

template <uint32_t kAct>
__device__ __forceinline__ void values8(floatx8& z) {
#pragma unroll
    for (int r = 0; r < 8; ++r) z[r] = act_value<kAct>(z[r]);
}
template <uint32_t kAct>
__device__ __forceinline__ void slopes8(floatx8& z) {
#pragma unroll
    for (int r = 0; r < 8; ++r) z[r] = act_slope<kAct>(z[r]);
}
__device__ __forceinline__ void act_values(uint32_t act, floatx8& z) {
    switch (act) {
    case NERF_EXT_ACT_RELU: return values8<NERF_EXT_ACT_RELU>(z);
    case NERF_EXT_ACT_SOFTPLUS: return values8<NERF_EXT_ACT_SOFTPLUS>(z);
    case NERF_EXT_ACT_SIGMOID: return values8<NERF_EXT_ACT_SIGMOID>(z);
    case NERF_EXT_ACT_SILU: return values8<NERF_EXT_ACT_SILU>(z);
    case NERF_EXT_ACT_GELU: return values8<NERF_EXT_ACT_GELU>(z);
    default: return;
    }
}
__device__ __forceinline__ void act_slopes(uint32_t act, floatx8& z) {
    switch (act) {
    case NERF_EXT_ACT_RELU: return slopes8<NERF_EXT_ACT_RELU>(z);
    case NERF_EXT_ACT_SOFTPLUS: return slopes8<NERF_EXT_ACT_SOFTPLUS>(z);
    case NERF_EXT_ACT_SIGMOID: return slopes8<NERF_EXT_ACT_SIGMOID>(z);
    case NERF_EXT_ACT_SILU: return slopes8<NERF_EXT_ACT_SILU>(z);
    case NERF_EXT_ACT_GELU: return slopes8<NERF_EXT_ACT_GELU>(z);
    default: return slopes8<NERF_EXT_ACT_NONE>(z);
    }
}

// Eight values of which `some` are an operand's, fetched from `down` values
// ahead of them: those moved to the front, zeros behind them.
__device__ __forceinline__ uint4 settled(uint4 v, uint32_t down, uint32_t some) {
    unsigned long long w[2];
    __builtin_memcpy(w, &v, 16);
    const uint32_t bits = 16u * (down & 3u);
    if (down >= 4u) {
        w[0] = w[1];
        w[1] = 0ull;
    }
    if (bits) {
        w[0] = w[0] >> bits | w[1] << (64u - bits);
        w[1] >>= bits;
    }
    const unsigned long long ones = ~0ull;
    w[0] &= some >= 4u ? ones : ~(ones << (16u * some));
    w[1] &= some >= 8u ? ones : some > 4u ? ~(ones << (16u * (some - 4u))) : 0ull;
    __builtin_memcpy(&v, w, 16);
    return v;
}

// ------------------------------------------------------------- epilogues
// What becomes of a finished sum.  Arrays are reached through buffer
// descriptors that start at the workgroup's first row: offsets are 32 bits,
// and an access whose offset is kBeyond does nothing (loads give 0), which
// takes the place of branches at the edges.
constexpr uint32_t kBeyond = 0x80000000u;
typedef unsigned int uintx4 __attribute__((ext_vector_type(4)));

template <typename E>
struct Rows {
    const E* base;
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t ld;
    // Row `first` of an array with rows ld elements apart.
    __device__ __forceinline__ Rows(const void* data, uint64_t first, uint64_t ld_) : base((const E*)data + first * ld_), rsrc(__builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)0x7FFFFFFF, 0x00020000)), ld((uint32_t)ld_) {}
    __device__ __forceinline__ uint32_t at(uint32_t row, uint32_t p) const { return (row * ld + p) * (uint32_t)sizeof(E); }
    // Eight elements from (row, p), n of them inside; vec: all or none, aligned to
    // 16 bytes.  Else (rows of at least eight) a lane with fewer fetches the eight
    // that end with its row, and widen() moves them: every lane by the same load,
    // since one that only some lanes take is waited for where they meet.
    __device__ __forceinline__ uintx4 load(uint32_t row, uint32_t p, uint32_t n, bool vec, bool rows_of_eight) const {
        static_assert(sizeof(E) == 2);
        if (vec) return __builtin_bit_cast(uintx4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(n ? at(row, p) : kBeyond), 0, 0));
        uintx4 o;
        if (rows_of_eight) {
            __builtin_memcpy(&o, base + (n ? row * ld + p + n - 8u : 0u), 16);
        } else {
            short8_t v;
#pragma unroll
            for (uint32_t r = 0; r < 8u; ++r) v[r] = (short)__builtin_amdgcn_raw_buffer_load_b16(rsrc, (int)(r < n ? at(row, p + r) : kBeyond), 0, 0);
            o = __builtin_bit_cast(uintx4, v);
        }
        return o;
    }
    __device__ __forceinline__ void store(uint32_t row, uint32_t p, uint32_t n, bool vec, const floatx8& v) const {
        if constexpr (sizeof(E) == 4) {
            // Copies: a bit cast of part of a vector takes the vector's first part.
            const floatx4 lo = v.lo, hi = v.hi;
            if (vec) {
                const uint32_t o = n ? at(row, p) : kBeyond;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, lo), rsrc, (int)o, 0, 0);
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, hi), rsrc, (int)(o + 16u), 0, 0);
            } else if (n == 8u) {
                __builtin_memcpy((void*)(base + row * ld + p), &lo, 16);
                __builtin_memcpy((void*)(base + row * ld + p + 4u), &hi, 16);
            } else if (n) {
#pragma unroll
                for (uint32_t r = 0; r < 8u; ++r) {
                    const float e = v[r];
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, e), rsrc, (int)(r < n ? at(row, p + r) : kBeyond), 0, 0);
                }
            }
        } else {
            const typename Vec<E>::x8 h = __builtin_convertvector(v, typename Vec<E>::x8);
            if (vec) {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, h), rsrc, (int)(n ? at(row, p) : kBeyond), 0, 0);
            } else if (n == 8u) {
                __builtin_memcpy((void*)(base + row * ld + p), &h, 16);
            } else if (n) {
                const short8_t b = __builtin_bit_cast(short8_t, h);
#pragma unroll
                for (uint32_t r = 0; r < 8u; ++r) __builtin_amdgcn_raw_buffer_store_b16(b[r], rsrc, (int)(r < n ? at(row, p + r) : kBeyond), 0, 0);
            }
        }
    }
};

// What Rows::load has fetched, as 32-bit values.
template <typename T>
__device__ __forceinline__ floatx8 widen(uintx4 v, uint32_t n, bool vec, bool rows_of_eight) {
    if (!vec && rows_of_eight) v = __builtin_bit_cast(uintx4, settled(__builtin_bit_cast(uint4, v), 8u - n, n));
    return __builtin_convertvector(__builtin_bit_cast(typename Vec<T>::x8, v), floatx8);
}

// The biases of p0 .. p0 + kB in LDS, zeros where there are none, and eight of
// them.  Loads return in their order: a bias loaded from memory as it is used
// is waited for with everything that was asked for before it, which was the
// next rows' operands (2^18 x 256 -> 256: 169 us with it, 117 us without).
// One bias a thread: asked for first and kept once the operands are asked for.
template <uint32_t kB, typename Out>
__device__ __forceinline__ float thread_bias(const Out& out, uint32_t p0) {
    if constexpr (Out::kBias)
        if (out.bias && threadIdx.x < kB && p0 + threadIdx.x < out.np) return out.bias[p0 + threadIdx.x];
    return 0.0f;
}
template <typename Out>
__device__ __forceinline__ floatx8 bias8(const float* lds, uint32_t at) {
    floatx8 b = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (Out::kBias) {
        b.lo = *reinterpret_cast<const floatx4*>(lds + at);
        b.hi = *reinterpret_cast<const floatx4*>(lds + at + 4u);
    }
    return b;
}

// Each epilogue gets eight consecutive p of one row q0 + row at a time, n of
// them inside the output (0 for a row outside), with their biases, and first
// loads what else it needs, so that a caller can have that under way early.
template <typename T>
struct ForwardOut {
    const float* bias;
    const T* residual;
    void* y;
    T* pre;
    uint64_t ldr, ldy;
    uint32_t np, nq, act;
    bool y32, vec;
    struct Aux {
        uintx4 residual;
    };
    static constexpr bool kBias = true;

    __device__ __forceinline__ Aux load(uint32_t q0, uint32_t row, uint32_t p, uint32_t n) const {
        return {residual ? Rows<T>(residual, q0, ldr).load(row, p, n, vec, np >= 8u) : uintx4{0u, 0u, 0u, 0u}};
    }
    __device__ __forceinline__ void put(uint32_t q0, uint32_t row, uint32_t p, uint32_t n, floatx8 z, const floatx8& b, const Aux& a) const {
        z += b;
        if (pre) Rows<T>(pre, q0, np).store(row, p, n, vec, z);
        act_values(act, z);
        if (residual) z += widen<T>(a.residual, n, vec, np >= 8u);
        if (y32) Rows<float>(y, q0, ldy).store(row, p, n, vec, z);
        else Rows<T>(y, q0, ldy).store(row, p, n, vec, z);
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
    struct Aux {
        uintx4 add, pre;
    };
    static constexpr bool kBias = false;

    __device__ __forceinline__ Aux load(uint32_t q0, uint32_t row, uint32_t p, uint32_t n) const {
        Aux a{};
        if (add) a.add = Rows<T>(add, q0, ldx).load(row, p, n, vec, np >= 8u);
        if (dpre) a.pre = Rows<T>(pre, q0, np).load(row, p, n, vec, np >= 8u);
        return a;
    }
    __device__ __forceinline__ void put(uint32_t q0, uint32_t row, uint32_t p, uint32_t n, floatx8 g, const floatx8&, const Aux& a) const {
        if (add) g += widen<T>(a.add, n, vec, np >= 8u);
        if (dx) Rows<T>(dx, q0, ldx).store(row, p, n, vec, g);
        if (dpre) {
            floatx8 s = widen<T>(a.pre, n, vec, np >= 8u);
            act_slopes(act, s);
            Rows<T>(dpre, q0, np).store(row, p, n, vec, g * s);
        }
    }
};

// Plain sums in 32 bits: dW, or one part of a sum that was split over k.
struct SumOut {
    float* out;       // the first part, or all of it
    float* parts;     // the others
    uint64_t part;    // elements from one of them to the next
    float* row_sums;  // sum_k Q(q, k), or null; nq of them a part
    uint32_t np, nq;
    bool vec;
    struct Aux {};
    static constexpr bool kBias = false;
    __device__ __forceinline__ Aux load(uint32_t, uint32_t, uint32_t, uint32_t) const { return {}; }
    __device__ __forceinline__ void put(uint32_t q0, uint32_t row, uint32_t p, uint32_t n, const floatx8& v, const floatx8&, const Aux&) const { Rows<float>(out, q0, np).store(row, p, n, vec, v); }
};

// ----------------------------------------------------------------- product
constexpr uint32_t kBK = 64u;  // k per tile: two matrix instructions' worth

struct Operands {
    const void* p;
    const void* q;
    uint64_t ldp, ldq;  // elements between rows in memory
    uint32_t np, nq, nk;
    uint32_t k_split;   // k per part, a multiple of kBK
    uint32_t tiles_p, tiles_q;
};

// A tile of kB rows x 64 k lies in LDS in 16-byte chunks of 8 values, the
// chunk's place xor-ed with bits of its line so that the lanes that the LDS
// serves together fall on different banks.  k contiguous: row-major [kB][64],
// 8 lanes a turn, the 8 rows in 8 different places.  kT (row contiguous):
// k-major [64][kB]; 32 lanes of a transposing read are served together, k 0..3
// and 8..11 of 32 bytes each, which go to the 8 different places of 256 bytes
// (with kB = 64 the line's parity is one of the place's bits already).  With
// both groups of four k in the same four places half of the LDS' cycles were
// conflicts.
template <uint32_t kB, bool kT>
__device__ __forceinline__ constexpr uint32_t chunk_key(uint32_t line) {
    if (!kT) return line & 7u;
    if (kB >= 128u) return ((line & 3u) | ((line >> 3) & 1u) << 2) << 1;
    return (((line >> 1) & 1u) | ((line >> 3) & 1u) << 1) << 1;
}
template <uint32_t kB, bool kT>
__device__ __forceinline__ constexpr uint32_t chunk_slot(uint32_t line, uint32_t chunk) {
    return line * (kT ? kB / 8u : 8u) + (chunk ^ chunk_key<kB, kT>(line));
}

// Eight values from any address.  The hardware serves 16 bytes that start at a
// multiple of 4 at full rate and others slowly (7 x 1601 -> 1000: 10.2 us with
// rows that start at odd values, 5.8 us at even ones), so operands whose rows
// may start at odd values (kWords) are fetched as the five 32-bit words that the
// values lie in, all of which hold some of them, and put together when they are
// used.
typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(4)));
template <bool kWords>
struct Eight {
    uint4 v;
    uint32_t fifth[kWords ? 1 : 0];

    template <typename T>
    __device__ __forceinline__ void fetch(const T* at) {
        if constexpr (kWords) {
            const uint32_t half = (uint32_t)((uintptr_t)at >> 1) & 1u;
            const word4 w       = *reinterpret_cast<const word4*>(at - half);
            v                   = uint4{w[0], w[1], w[2], w[3]};
            fifth[0]            = *reinterpret_cast<const uint32_t*>(at + 6u + half);
        } else {
            __builtin_memcpy(&v, at, 16);
        }
    }
    // place: the address' number of values, at least its last bit.
    __device__ __forceinline__ uint4 value(uint32_t place) const {
        if constexpr (kWords) {
            const uint32_t s = 16u * (place & 1u);
            return uint4{__builtin_amdgcn_alignbit(v.y, v.x, s), __builtin_amdgcn_alignbit(v.z, v.y, s), __builtin_amdgcn_alignbit(v.w, v.z, s), __builtin_amdgcn_alignbit(fifth[0], v.w, s)};
        }
        return v;
    }
};
// Number of an address in values, for Eight::value.
template <typename T>
__device__ __forceinline__ uint32_t value_number(const T* p) { return (uint32_t)((uintptr_t)p >> 1); }

// Where a lane finds eight values of an operand at its edges: from a place that
// ends with the line (or begins with the array, which has eight values at
// least), `some` of them the operand's, `down` values on.
struct Edge {
    uint64_t at;
    uint32_t some, down;
};
// line: the values' line (row, or k where rows are contiguous) of `lines`, minor
// their place in it, of `length`.
__device__ __forceinline__ Edge edge(uint64_t ld, uint32_t line, uint32_t lines, uint32_t minor, uint32_t length) {
    Edge e;
    e.some             = line < lines && minor < length ? min(8u, length - minor) : 0u;
    const uint64_t own = (uint64_t)line * ld + minor, end = own + e.some;
    e.at               = e.some && end > 8u ? end - 8u : 0ull;
    e.down             = e.some ? (uint32_t)(own - e.at) : 0u;
    return e;
}

// Tile [row0, row0 + kB) x [k0, k0 + 64) into LDS, zeros outside [0, n) x [0, k_end),
// through registers and at any alignment: fetch() asks for a tile, keep() writes
// it to LDS.  What differs at the edges is the addresses, before the loads, and
// keep(): a branch with a load in it, or an edge's work right behind its load,
// makes the loads wait for each other (20011 x 1209 -> 487 took 112 us).
template <typename T, uint32_t kB, bool kT, uint32_t kThreads, bool kWords>
struct Stager {
    static constexpr uint32_t kChunks = kT ? kB / 8u : 8u;
    static constexpr uint32_t kLoads  = kB * 8u / kThreads;
    static_assert(kB * 8u % kThreads == 0u);
    Eight<kWords> held[kLoads];

    static __device__ __forceinline__ uint32_t line(uint32_t i) { return (i * kThreads + threadIdx.x) / kChunks; }
    static __device__ __forceinline__ uint32_t chunk(uint32_t i) { return (i * kThreads + threadIdx.x) % kChunks; }
    static __device__ __forceinline__ bool inner(uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) { return row0 + kB <= n && k0 + kBK <= k_end; }
    static __device__ __forceinline__ Edge place(uint32_t i, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) {
        return kT ? edge(ld, k0 + line(i), k_end, row0 + 8u * chunk(i), n) : edge(ld, row0 + line(i), n, k0 + 8u * chunk(i), k_end);
    }

    __device__ __forceinline__ void fetch(const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) {
        uint64_t at[kLoads];
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) at[i] = (uint64_t)((kT ? k0 : row0) + line(i)) * ld + (kT ? row0 : k0) + 8u * chunk(i);
        if (!inner(n, row0, k0, k_end)) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) at[i] = place(i, ld, n, row0, k0, k_end).at;
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) held[i].fetch(src + at[i]);
    }
    __device__ __forceinline__ void keep(uint4* lds, const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) const {
        const uint32_t first = value_number(src);
        if (inner(n, row0, k0, k_end)) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) lds[chunk_slot<kB, kT>(line(i), chunk(i))] = held[i].value(first + ((kT ? k0 : row0) + line(i)) * (uint32_t)ld + (kT ? row0 : k0));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const Edge e                                 = place(i, ld, n, row0, k0, k_end);
                lds[chunk_slot<kB, kT>(line(i), chunk(i))] = settled(held[i].value(first + (uint32_t)e.at), e.down, e.some);
            }
        }
    }
};

// The same straight from memory into LDS, 16 bytes a lane, for chunks that are
// whole and aligned (start, stride and the contiguous length multiples of 8):
// a wave fills 64 slots in their order, each lane fetching the chunk whose
// place its slot is.  Chunks outside the operand take an offset beyond the
// descriptor's range, for which the hardware delivers zeros.
template <typename T, uint32_t kB, bool kT, uint32_t kThreads>
struct Loader {
    static constexpr uint32_t kChunks = kT ? kB / 8u : 8u;
    static constexpr uint32_t kLoads  = kB * 8u / kThreads;
    static_assert(kB * 8u % kThreads == 0u);
    const T* base;           // of the tile at its next k
    uint64_t step;           // elements from one tile of k to the next
    uint32_t offset[kLoads]; // bytes, kBeyond for rows outside
    uint32_t minor;          // kT: unused; else the lane's first k within the tile

    __device__ __forceinline__ void begin(const T* src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0) {
        base = src + (kT ? (uint64_t)k0 * ld + row0 : (uint64_t)row0 * ld + k0);
        step = kT ? kBK * ld : kBK;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t s = i * kThreads + threadIdx.x, line = s / kChunks, chunk = (s % kChunks) ^ chunk_key<kB, kT>(line);
            const bool inside = kT ? row0 + 8u * chunk < n : row0 + line < n;
            offset[i]         = inside ? (line * (uint32_t)ld + 8u * chunk) * 2u : kBeyond;
        }
    }
    // left: k from the tile's start to the end of the part.
    __device__ __forceinline__ void issue(uint4* lds, int left) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)0x7FFFFFFF, 0x00020000);
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            uint32_t at = offset[i];
            if (left < (int)kBK) {
                const uint32_t s = i * kThreads + threadIdx.x, line = s / kChunks, chunk = (s % kChunks) ^ chunk_key<kB, kT>(line);
                if ((int)(kT ? line : 8u * chunk) >= left) at = kBeyond;
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + i * kThreads + wave * 64u), 16, (int)at, 0, 0, 0);
        }
        base += step;
    }
};

// The 8 k of 16 rows that a lane feeds to one 16x16x32 matrix instruction:
// k = 32 step + 8 (lane / 16) + 0..7 of row wave0 + 16 i + lane % 16.  A lane
// keeps one place in a tile (fragment_base: i = step = 0); the others differ
// from it by constants and by single bits, which are put in as they are used
// (held in registers, the places of all fragments left too few for the sums).
template <uint32_t kB, bool kT>
__device__ __forceinline__ uint32_t fragment_base(uint32_t wave0) {
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, g = lane >> 4;
    if (!kT) return 16u * chunk_slot<kB, false>(wave0 + l, g);
    const uint32_t row = wave0 + 4u * (l & 3u);
    return 16u * chunk_slot<kB, true>(8u * g + (l >> 2), row >> 3) + 2u * (row & 7u);
}
template <typename T, uint32_t kB, bool kT>
__device__ __forceinline__ typename Vec<T>::x8 fragment(const uint4* lds, uint32_t base, uint32_t i, uint32_t step) {
    const char* tile = reinterpret_cast<const char*>(lds);
    if constexpr (!kT) {
        return *reinterpret_cast<const typename Vec<T>::x8*>(tile + (base ^ (64u * step)) + 2048u * i);
    } else {
        // Lane 4 r + c of 16 reads rows 4 c .. 4 c + 3 at k = r; the read hands lane
        // l the four k of row l.
        short4_t h[2];
#pragma unroll
        for (uint32_t half = 0; half < 2u; ++half) h[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(tile + (base ^ (32u * i)) + 2u * kB * (32u * step + 4u * half)));
        return __builtin_bit_cast(typename Vec<T>::x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// Has a fragment in registers here.  The compiler moves a transposing read that
// is used behind a barrier to behind it, where its LDS is written again.
template <typename V>
__device__ __forceinline__ void settle_here(V& v) {
    asm volatile("" : "+v"(v)::"memory");
}

// Waits until at most `kLater` of the wave's own loads are on their way, and
// then for the workgroup.
template <uint32_t kLater>
__device__ __forceinline__ void arrived() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (kLater & 15u) | (kLater >> 4) << 14);  // vmcnt
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The card gives workgroups to its eight chips in turn, each with an L2 of its
// own.  Tile number of workgroup b of n, so that a chip's workgroups have tiles in
// a row: those share operands.
__device__ __forceinline__ uint32_t chip_tile(uint32_t b, uint32_t n) {
    const uint32_t chip = b % 8u, each = n / 8u, more = n % 8u;
    return chip * each + min(chip, more) + b / 8u;
}

// out(q, p) = sum_k P(p, k) Q(q, k), kBP x kBQ outputs a workgroup, kWP x kWQ
// waves, kDepth tiles of 64 k at a time in LDS or on their way there.  kMode: both
// operands go straight into LDS (kDirect), or the tiles on their way wait in
// registers, fetched by chunks or as words.
// The matrix cores bound it where the outputs are wide: a wave of the 256 tile has
// 128 x 64 sums in registers and reads 192 rows of k from LDS for them (without
// bank conflicts), 16384 x 4096 -> 4096 in bf16 470 us = 1.17 PFLOP/s, where a
// library's product alone reaches 1.24.  Four buffers of 32 k there, with the next
// tile's first fragments read a barrier ahead, took 493.  Where they are narrow the
// memory does: the weights' gradient of 262144 x 256 -> 256 69 us = 3.9 TB/s.
enum Mode : uint32_t { kDirect, kByChunks, kByWords };
template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, uint32_t kDepth, bool kPT, bool kQT, Mode kMode, typename Out>
__global__ __launch_bounds__(kWP * kWQ * 64u) void k_product(Operands A, Out out) {
    constexpr uint32_t kThreads = kWP * kWQ * 64u;
    constexpr uint32_t kFP = kBP / kWP / 16u, kFQ = kBQ / kWQ / 16u;
    // Variables of their own, so that the compiler sees that a read of one is no
    // read of what is on its way into another.
    constexpr bool kAligned  = kMode == kDirect;
    constexpr uint32_t kTile = (kBP + kBQ) * 8u;
    static_assert(!kAligned || kDepth == 2u || kDepth == 4u);
    __shared__ uint4 lds0[kTile], lds1[kAligned ? kTile : 1u], lds2[kAligned && kDepth == 4u ? kTile : 1u], lds3[kAligned && kDepth == 4u ? kTile : 1u];
    __shared__ floatx4 lds_bias[Out::kBias ? kBP / 4u : 1u];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t wp = (wave % kWP) * (kBP / kWP), wq = (wave / kWP) * (kBQ / kWQ);
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

    // Sums of Q over k, for out.row_sums: a product with ones, the fragments of Q
    // shared out among the waves that hold the same.
    constexpr bool kSums = std::is_same_v<Out, SumOut>;
    constexpr uint32_t kSumsQ = kSums ? kFQ / kWP : 1u;
    static_assert(kBP <= kThreads);
    const float bias = thread_bias<kBP>(out, p0);
    auto keep_bias   = [&] {
        if (Out::kBias && threadIdx.x < kBP) reinterpret_cast<float*>(lds_bias)[threadIdx.x] = bias;
    };
    floatx4 acc[kFP][kFQ], sums[kSumsQ];
#pragma unroll
    for (uint32_t j = 0; j < kSumsQ; ++j) sums[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t j = 0; j < kFQ; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < kFP; ++i) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bool take_sums = false;
    if constexpr (kSums) take_sums = out.row_sums && tile_p == 0u;
    typename Vec<T>::x8 ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = (T)1.0f;

    const uint32_t base_p = fragment_base<kBP, kPT>(wp), base_q = fragment_base<kBQ, kQT>(wq);
    // One tile of 64 k: kG fragments of P against all of Q at a time, the next
    // fragments on their way from LDS meanwhile.
    constexpr uint32_t kG = kFP < 2u ? 1u : 2u, kPhases = kFP / kG;
    auto multiply = [&](const uint4* lp) {
        const uint4* lq = lp + kBP * 8u;
        typename Vec<T>::x8 fp[2][kG], fq[2][kFQ];
        uint32_t bp = base_p, bq = base_q;
        asm volatile("" : "+v"(bp), "+v"(bq));
        auto fetch_p = [&](uint32_t phase) {
#pragma unroll
            for (uint32_t g = 0; g < kG; ++g) fp[phase & 1u][g] = fragment<T, kBP, kPT>(lp, bp, phase % kPhases * kG + g, phase / kPhases);
        };
        auto fetch_q = [&](uint32_t step) {
#pragma unroll
            for (uint32_t j = 0; j < kFQ; ++j) fq[step][j] = fragment<T, kBQ, kQT>(lq, bq, j, step);
        };
        fetch_q(0u);
        fetch_p(0u);
#pragma unroll
        for (uint32_t phase = 0; phase < 2u * kPhases; ++phase) {
            const uint32_t step = phase / kPhases;
            if (phase + 1u < 2u * kPhases) {
                if ((phase + 1u) % kPhases == 0u) fetch_q(step + 1u);
                fetch_p(phase + 1u);
            }
#pragma unroll
            for (uint32_t g = 0; g < kG; ++g)
#pragma unroll
                for (uint32_t j = 0; j < kFQ; ++j) acc[phase % kPhases * kG + g][j] = Vec<T>::mfma(fp[phase & 1u][g], fq[step][j], acc[phase % kPhases * kG + g][j]);
            if constexpr (kSums) {
                if (take_sums && phase % kPhases == 0u) {
#pragma unroll
                    for (uint32_t c = 0; c < kWP; ++c)
                        if (wave % kWP == c) {
#pragma unroll
                            for (uint32_t j = 0; j < kSumsQ; ++j) sums[j] = Vec<T>::mfma(ones, fq[step][c * kSumsQ + j], sums[j]);
                        }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if constexpr (kAligned) {
        Loader<T, kBP, kPT, kThreads> load_p;
        Loader<T, kBQ, kQT, kThreads> load_q;
        load_p.begin((const T*)A.p, A.ldp, A.np, p0, k0);
        load_q.begin((const T*)A.q, A.ldq, A.nq, q0, k0);
        constexpr uint32_t kLoads = kBP * 8u / kThreads + kBQ * 8u / kThreads;
        auto issue = [&](uint4* lds, int left) {
            load_p.issue(lds, left);
            load_q.issue(lds + kBP * 8u, left);
        };
        constexpr int kStep = (int)kBK;
        int left            = (int)(k_end - k0);
        if constexpr (kDepth == 2u) {
            // Two tiles a turn; a last odd tile is followed by one of zeros (a way out
            // between the two would keep a second copy of the sums alive).  arrived():
            // everyone's part of the tile has come, and everyone is done with the
            // other buffer.
            issue(lds0, left);
            keep_bias();
            for (; left > 0; left -= 2 * kStep) {
                arrived<0u>();
                issue(lds1, left - kStep);
                multiply(lds0);
                arrived<0u>();
                if (left > 2 * kStep) issue(lds0, left - 2 * kStep);
                multiply(lds1);
            }
        } else {
            // Three tiles on their way: few k are asked for all at once.
            issue(lds0, left);
            issue(lds1, left - kStep);
            issue(lds2, left - 2 * kStep);
            keep_bias();
            for (; left > 0; left -= 4 * kStep) {
                arrived<2u * kLoads>();
                issue(lds3, left - 3 * kStep);
                multiply(lds0);
                arrived<2u * kLoads>();
                issue(lds0, left - 4 * kStep);
                if (left > kStep) multiply(lds1);
                arrived<2u * kLoads>();
                issue(lds1, left - 5 * kStep);
                if (left > 2 * kStep) multiply(lds2);
                arrived<2u * kLoads>();
                issue(lds2, left - 6 * kStep);
                if (left > 3 * kStep) multiply(lds3);
            }
        }
    } else {
        // The next kDepth - 1 tiles wait in registers.
        Stager<T, kBP, kPT, kThreads, kMode == kByWords> stage_p[kDepth - 1u];
        Stager<T, kBQ, kQT, kThreads, kMode == kByWords> stage_q[kDepth - 1u];
        auto fetch = [&](uint32_t d, uint32_t k) {
            stage_p[d].fetch((const T*)A.p, A.ldp, A.np, p0, k, k_end);
            stage_q[d].fetch((const T*)A.q, A.ldq, A.nq, q0, k, k_end);
        };
#pragma unroll
        for (uint32_t d = 0; d < kDepth - 1u; ++d)
            if (k0 + kBK * d < k_end) fetch(d, k0 + kBK * d);
        keep_bias();
        for (uint32_t k = k0; k < k_end; k += kBK * (kDepth - 1u)) {
#pragma unroll
            for (uint32_t d = 0; d < kDepth - 1u; ++d) {
                const uint32_t kd = k + kBK * d;
                if (kd < k_end) {
                    stage_p[d].keep(lds0, (const T*)A.p, A.ldp, A.np, p0, kd, k_end);
                    stage_q[d].keep(lds0 + kBP * 8u, (const T*)A.q, A.ldq, A.nq, q0, kd, k_end);
                    __syncthreads();
                    if (kd + kBK * (kDepth - 1u) < k_end) fetch(d, kd + kBK * (kDepth - 1u));
                    multiply(lds0);
                    __syncthreads();
                }
            }
        }
    }

    if constexpr (std::is_same_v<Out, SumOut>) {
        if (part) out.out = out.parts + (part - 1u) * out.part;
        if (take_sums && lane < 16u) {  // every p of the product with ones holds the sum
#pragma unroll
            for (uint32_t j = 0; j < kSumsQ; ++j) {
                const uint32_t q = q0 + wq + 16u * (wave % kWP * kSumsQ + j) + lane;
                if (q < out.nq) out.row_sums[(uint64_t)part * out.nq + q] = sums[j][0];
            }
        }
    }

    // The wave's sums, 16 q x kSP p at a time, through LDS of its own into rows:
    // a lane then has eight consecutive p, and eight lanes one 128-byte line
    // (16-bit outputs).  Chunks of four p, their place xor-ed with the row.
    constexpr uint32_t kSP = kBP / kWP < 64u ? kBP / kWP : 64u, kStrips = kFQ * (kBP / kWP / kSP);
    constexpr uint32_t kLanes = kSP / 8u, kPasses = 16u * kLanes / 64u;
    static_assert(kWP * kWQ * kSP * 4u <= kTile);
    __syncthreads();
    arrived<0u>();  // the zeros behind the last tile too
    floatx4* strip = reinterpret_cast<floatx4*>(lds0) + wave * (kSP * 4u);
    const uint32_t row = lane / kLanes, col = 8u * (lane % kLanes);
    auto row_of = [&](uint32_t s, uint32_t pass) { return wq + 16u * (s % kFQ) + (64u / kLanes) * pass + row; };
    auto p_of = [&](uint32_t s) { return p0 + wp + kSP * (s / kFQ) + col; };
    auto inside = [&](uint32_t s, uint32_t pass) { return q0 + row_of(s, pass) < out.nq && p_of(s) < out.np ? min(8u, out.np - p_of(s)) : 0u; };
    typename Out::Aux aux[2][kPasses];
    auto prefetch = [&](uint32_t s) {
#pragma unroll
        for (uint32_t t = 0; t < kPasses; ++t) aux[s & 1u][t] = out.load(q0, row_of(s, t), p_of(s), inside(s, t));
    };
    prefetch(0u);
#pragma unroll
    for (uint32_t s = 0; s < kStrips; ++s) {
#pragma unroll
        for (uint32_t f = 0; f < kSP / 16u; ++f) strip[(lane & 15u) * (kSP / 4u) + ((4u * f + (lane >> 4)) ^ (lane & 7u))] = acc[kSP / 16u * (s / kFQ) + f][s % kFQ];
        if (s + 1u < kStrips) prefetch(s + 1u);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (uint32_t t = 0; t < kPasses; ++t) {
            const uint32_t r = (64u / kLanes) * t + row;
            floatx8 v;
            v.lo = strip[r * (kSP / 4u) + ((col / 4u) ^ (r & 7u))];
            v.hi = strip[r * (kSP / 4u) + ((col / 4u + 1u) ^ (r & 7u))];
            out.put(q0, row_of(s, t), p_of(s), inside(s, t), v, bias8<Out>(reinterpret_cast<const float*>(lds_bias), p_of(s) - p0), aux[s & 1u][t]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
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
constexpr uint32_t kStreamWaves = 8u;
template <typename T, uint32_t kKS, uint32_t kFP, bool kPT, bool kRagged, bool kWords, typename Out>
__global__ __launch_bounds__(kStreamWaves * 64u) void k_stream(Operands A, Out out, uint32_t p_waves) {
    // Where P takes half of the registers, the outputs' edges have to do without any.
    if constexpr (kKS * kFP == 32u) out.vec = true;
    constexpr uint32_t kThreads = kStreamWaves * 64u, kSP = 16u * kFP, kBP = 256u;
    constexpr uint32_t kLanes = kSP / 8u, kPasses = 16u * kLanes / 64u;
    using x8 = typename Vec<T>::x8;
    __shared__ uint4 lds[kBP * 8u];
    __shared__ floatx4 lds_bias[Out::kBias ? kBP / 4u : 1u];
    static_assert(kStreamWaves * kSP * 4u <= kBP * 8u);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t wp = wave % p_waves * kSP, p0 = blockIdx.y * p_waves * kSP;

    x8 fp[kKS][kFP];
    {
        const float bias = thread_bias<kBP>(out, p0);
        Stager<T, kBP, kPT, kThreads, true> stager;
        stager.fetch((const T*)A.p, A.ldp, A.np, p0, 0u, A.nk);
        if (Out::kBias && threadIdx.x < kBP) reinterpret_cast<float*>(lds_bias)[threadIdx.x] = bias;
        const uint32_t base = fragment_base<kBP, kPT>(wp & ~127u);
#pragma unroll
        for (uint32_t s = 0; s < kKS; s += 2u) {
            stager.keep(lds, (const T*)A.p, A.ldp, A.np, p0, 32u * s, A.nk);
            __syncthreads();
            if (s + 2u < kKS) stager.fetch((const T*)A.p, A.ldp, A.np, p0, 32u * (s + 2u), A.nk);
#pragma unroll
            for (uint32_t i = 0; i < kFP; ++i)
#pragma unroll
                for (uint32_t h = 0; h < 2u; ++h)
                    if (s + h < kKS) {
                        fp[s + h][i] = fragment<T, kBP, kPT>(lds, base, (wp & 127u) / 16u + i, h);
                        settle_here(fp[s + h][i]);
                    }
            __syncthreads();
        }
    }

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

// --------------------------------------------------------------- few tiles
// Products of too few outputs to occupy the card by tiles: what counts is the
// time of one workgroup and the number of launches.  A workgroup has a tile of
// 16 kF x 16 kF outputs, its eight waves every eighth 32 k each; a wave fetches
// its operands from memory itself, several steps at a time and without waiting
// for the others, and the eight sums are added in LDS in their order.  (A
// launch costs the host 3.5 us, about what such a kernel takes; one with 64 x 64
// tiles whose k were split over workgroups and a second one to join them took
// 12 us for 7 x 1601 -> 999, this one 7; backward 37 x 788 -> 64 4 us, in three
// launches 10.)
constexpr uint32_t kFewWaves = 8u;

// 16 kF rows x 32 k of an operand, any alignment, on its way to one wave; the
// edges as Stager has them.  Rows outside are other rows: their products are in
// outputs that nothing reads.
template <typename T, uint32_t kF, bool kT, bool kWords>
struct FewOperand {
    using x8 = typename Vec<T>::x8;
    static constexpr uint32_t kChunks = 2u * kF;  // of a line of 16 kF rows (kT)
    Eight<kWords> held[kF];

    static __device__ __forceinline__ uint64_t own(uint32_t i, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0) {
        const uint32_t lane = threadIdx.x & 63u;
        if (kT) return (uint64_t)(k0 + (i * 64u + lane) / kChunks) * ld + row0 + 8u * ((i * 64u + lane) % kChunks);
        return (uint64_t)min(row0 + 16u * i + (lane & 15u), n - 1u) * ld + k0 + 8u * (lane >> 4);
    }
    static __device__ __forceinline__ Edge place(uint32_t i, uint64_t ld, uint32_t n, uint32_t nk, uint32_t row0, uint32_t k0) {
        const uint32_t lane = threadIdx.x & 63u;
        if (kT) return edge(ld, k0 + (i * 64u + lane) / kChunks, nk, row0 + 8u * ((i * 64u + lane) % kChunks), n);
        return edge(ld, min(row0 + 16u * i + (lane & 15u), n - 1u), n, k0 + 8u * (lane >> 4), nk);
    }
    static __device__ __forceinline__ bool inner(uint32_t n, uint32_t nk, uint32_t row0, uint32_t k0) { return k0 + 32u <= nk && (!kT || row0 + 16u * kF <= n); }

    __device__ __forceinline__ void fetch(const Operands& A, const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0) {
        uint64_t at[kF];
#pragma unroll
        for (uint32_t i = 0; i < kF; ++i) at[i] = own(i, ld, n, row0, k0);
        if (!inner(n, A.nk, row0, k0)) {
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) at[i] = place(i, ld, n, A.nk, row0, k0).at;
        }
#pragma unroll
        for (uint32_t i = 0; i < kF; ++i) held[i].fetch(src + at[i]);
    }
    // The fragments of what was fetched; lds: 1024 kF bytes of the wave's own (kT).
    __device__ __forceinline__ void take(const Operands& A, const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, char* lds, x8 out[kF]) {
        const uint32_t first = value_number(src);
        uint4 v[kF];
        if (inner(n, A.nk, row0, k0)) {
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) v[i] = held[i].value(first + (uint32_t)own(i, ld, n, row0, k0));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) {
                const Edge e = place(i, ld, n, A.nk, row0, k0);
                v[i]         = settled(held[i].value(first + (uint32_t)e.at), e.down, e.some);
            }
        }
        if constexpr (!kT) {
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) out[i] = __builtin_bit_cast(x8, v[i]);
        } else {
            const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, g = lane >> 4;
            auto slot = [](uint32_t line, uint32_t chunk) { return line * kChunks + (chunk ^ (kF == 4u ? chunk_key<64u, true>(line) : 0u)); };
            asm volatile("" ::: "memory");
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) reinterpret_cast<uint4*>(lds)[slot((i * 64u + lane) / kChunks, (i * 64u + lane) % kChunks)] = v[i];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) {
                short4_t h[2];
#pragma unroll
                for (uint32_t half = 0; half < 2u; ++half) {
                    const uint32_t row = 16u * i + 4u * (l & 3u);
                    h[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(lds + 16u * slot(8u * g + 4u * half + (l >> 2), row >> 3) + 2u * (row & 7u)));
                }
                out[i] = __builtin_bit_cast(x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) settle_here(out[i]);
        }
    }
};

constexpr uint32_t few_lds(uint32_t f) { return kFewWaves * std::max(16u * f * 16u * f * 4u, 2048u * f); }

template <typename T, uint32_t kF, bool kPT, bool kQT, bool kWords, typename Out>
__device__ __forceinline__ void few_tile(const Operands& A, const Out& out, uint32_t p0, uint32_t q0, char* lds, float* lds_sums) {
    constexpr bool kSums = std::is_same_v<Out, SumOut>;
    constexpr uint32_t kDepth = kF == 1u ? 8u : kF == 2u ? 3u : 2u;  // steps on their way
    constexpr uint32_t kSP = 16u * kF, kEights = 16u * kF * kSP / 8u;
    using x8 = typename Vec<T>::x8;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;

    // What the outputs need besides the sums: the thread's eight outputs.
    const uint32_t row = threadIdx.x / (kSP / 8u), col = 8u * (threadIdx.x % (kSP / 8u)), p = p0 + col;
    const uint32_t n = threadIdx.x < kEights && q0 + row < out.nq && p < out.np ? min(8u, out.np - p) : 0u;
    floatx8 bias = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (Out::kBias) {
        if (out.bias) {
#pragma unroll
            for (uint32_t r = 0; r < 8u; ++r) bias[r] = r < n ? out.bias[p + r] : 0.0f;
        }
    }
    const typename Out::Aux aux = out.load(q0, row, p, n);

    floatx4 acc[kF][kF], sums[kF];
#pragma unroll
    for (uint32_t j = 0; j < kF; ++j) {
        sums[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t i = 0; i < kF; ++i) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const bool take_sums = kSums && p0 == 0u;
    x8 ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = (T)1.0f;
    FewOperand<T, kF, kPT, kWords> op[kDepth];
    FewOperand<T, kF, kQT, kWords> oq[kDepth];
    char* mine = lds + wave * 2048u * kF;
    auto fetch = [&](uint32_t d, uint32_t k) {
        op[d].fetch(A, (const T*)A.p, A.ldp, A.np, p0, k);
        oq[d].fetch(A, (const T*)A.q, A.ldq, A.nq, q0, k);
    };
    constexpr uint32_t kStride = 32u * kFewWaves;
#pragma unroll
    for (uint32_t d = 0; d < kDepth; ++d)
        if (32u * wave + kStride * d < A.nk) fetch(d, 32u * wave + kStride * d);
    for (uint32_t k = 32u * wave; k < A.nk; k += kStride * kDepth) {
#pragma unroll
        for (uint32_t d = 0; d < kDepth; ++d) {
            const uint32_t kd = k + kStride * d;
            if (kd < A.nk) {
                x8 fp[kF], fq[kF];
                op[d].take(A, (const T*)A.p, A.ldp, A.np, p0, kd, mine, fp);
                oq[d].take(A, (const T*)A.q, A.ldq, A.nq, q0, kd, mine + 1024u * kF, fq);
                if (kd + kStride * kDepth < A.nk) fetch(d, kd + kStride * kDepth);
#pragma unroll
                for (uint32_t i = 0; i < kF; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < kF; ++j) acc[i][j] = Vec<T>::mfma(fp[i], fq[j], acc[i][j]);
                if (take_sums) {
#pragma unroll
                    for (uint32_t j = 0; j < kF; ++j) sums[j] = Vec<T>::mfma(ones, fq[j], sums[j]);
                }
            }
        }
    }

    __syncthreads();  // the waves' own pieces become those of the sums
    floatx4* strips = reinterpret_cast<floatx4*>(lds);
    constexpr uint32_t kStrip = 16u * kF * kSP / 4u;
#pragma unroll
    for (uint32_t j = 0; j < kF; ++j) {
        const uint32_t r = 16u * j + (lane & 15u);
#pragma unroll
        for (uint32_t i = 0; i < kF; ++i) strips[wave * kStrip + r * (kSP / 4u) + ((4u * i + (lane >> 4)) ^ (r & 3u))] = acc[i][j];
        if (take_sums && lane < 16u) lds_sums[wave * 16u * kF + r] = sums[j][0];
    }
    __syncthreads();
    if (threadIdx.x < kEights) {
        floatx8 v = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < kFewWaves; ++w) {
            v.lo += strips[w * kStrip + row * (kSP / 4u) + ((col / 4u) ^ (row & 3u))];
            v.hi += strips[w * kStrip + row * (kSP / 4u) + ((col / 4u + 1u) ^ (row & 3u))];
        }
        out.put(q0, row, p, n, v, bias, aux);
    }
    if constexpr (kSums) {
        if (take_sums && out.row_sums && threadIdx.x < 16u * kF && q0 + threadIdx.x < out.nq) {
            float v = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kFewWaves; ++w) v += lds_sums[w * 16u * kF + threadIdx.x];
            out.row_sums[q0 + threadIdx.x] = v;
        }
    }
}

template <typename T, uint32_t kF, bool kWords>
__global__ __launch_bounds__(kFewWaves * 64u) void k_few_forward(Operands A, ForwardOut<T> out) {
    __shared__ floatx4 lds[few_lds(kF) / 16u];
    few_tile<T, kF, false, false, kWords>(A, out, blockIdx.x * 16u * kF, blockIdx.y * 16u * kF, reinterpret_cast<char*>(lds), nullptr);
}

// Both gradients in one launch: first the tiles of dx, x_tiles across and
// x_blocks in all, then those of dW.
template <typename T, uint32_t kF, bool kWords>
__global__ __launch_bounds__(kFewWaves * 64u) void k_few_backward(Operands X, InputGradientOut<T> x_out, uint32_t x_tiles, uint32_t x_blocks, Operands W, SumOut w_out, uint32_t w_tiles) {
    __shared__ floatx4 lds[few_lds(kF) / 16u];
    __shared__ float lds_sums[kFewWaves * 16u * kF];
    if (blockIdx.x < x_blocks) {
        few_tile<T, kF, true, false, kWords>(X, x_out, blockIdx.x % x_tiles * 16u * kF, blockIdx.x / x_tiles * 16u * kF, reinterpret_cast<char*>(lds), nullptr);
    } else {
        const uint32_t b = blockIdx.x - x_blocks;
        few_tile<T, kF, true, true, kWords>(W, w_out, b % w_tiles * 16u * kF, b / w_tiles * 16u * kF, reinterpret_cast<char*>(lds), lds_sums);
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
constexpr uint32_t kMaxFeatures = 1u << 16, kMaxStride = 1u << 20, kMaxRows = 1u << 30;

bool aligned(const void* p, uint64_t bytes) { return ((uintptr_t)p & (bytes - 1u)) == 0u; }
uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1u) / b); }

struct Workspace {
    float* data;
    uint64_t bytes;
};

// Whether an operand's rows may start at odd values.
bool odd_rows(const void* p, uint64_t ld) { return (((uintptr_t)p >> 1 | ld) & 1u) != 0u; }
// Whether an operand's chunks of 8 along its contiguous length are whole and aligned.
bool whole_chunks(const void* p, uint64_t ld, uint32_t contiguous) { return aligned(p, 16u) && ld % 8u == 0u && contiguous % 8u == 0u; }

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
constexpr uint32_t kFewMaxK = 4096u;
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
    if (d.x_stride > kMaxStride || d.y_stride > kMaxStride || d.residual_stride > kMaxStride) return refuse("a row stride is above 2^20");
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
