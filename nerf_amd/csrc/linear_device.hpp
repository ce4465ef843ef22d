// linear_device.hpp — what the kernels of linear layers share (linear.hip, and
// grouped.hip for layers with weights or adapters of many groups): types,
// activations, operands on their way from memory through LDS into the matrix
// instructions, and the two ways through a product, by tiles and by few tiles.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace nerf_hip {
namespace linear {

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
// ahead of them (at most eight in all): those moved to the front, zeros behind them.
// By 32-bit words: a 64-bit shift whose amount was in the last register of a wave's
// allocation has given wrong bits here now and then (tests/test_code_objects.py).
// What is behind them is multiplied by 0, two values at a time, else by 1 (20011 x 1209
// -> 487: 95 us, with comparisons and choices of each value 98).
__device__ __forceinline__ uint4 settled(uint4 v, uint32_t down, uint32_t some) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const uint32_t bits = 16u * (down & 1u);
    uint32_t w[4] = {__builtin_amdgcn_alignbit(v.y, v.x, bits), __builtin_amdgcn_alignbit(v.z, v.y, bits), __builtin_amdgcn_alignbit(v.w, v.z, bits), v.w >> bits};
    const bool one = down & 2u, two = down & 4u;
    w[0] = one ? w[1] : w[0];
    w[1] = one ? w[2] : w[1];
    w[2] = one ? w[3] : w[2];
    w[0] = two ? w[2] : w[0];
    w[1] = two ? w[3] : w[1];
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const u16x2 keep = __builtin_elementwise_min(__builtin_elementwise_sub_sat((u16x2)(unsigned short)some, u16x2{(unsigned short)(2u * i), (unsigned short)(2u * i + 1u)}), (u16x2)(unsigned short)1);
        w[i]             = __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, w[i]) * keep);
    }
    return uint4{w[0], w[1], w[2], w[3]};
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
constexpr uint32_t kStreamWaves = 8u;  // of the kernels that stream rows past weights in registers

struct Operands {
    const void* p;
    const void* q;
    uint64_t ldp, ldq;  // elements between rows in memory
    uint32_t np, nq, nk;
    uint32_t k_split;   // k per part, a multiple of kBK
    uint32_t tiles_p, tiles_q;
};

// Operands whose lines are rows in another order: Q's rows (forward, dx) or both
// operands' k (dW) are the rows that an index names, or themselves where it is
// null.  Rows at or beyond the count are zeros.
struct GatheredOperands : Operands {
    const uint32_t *p_index, *q_index;
    uint32_t p_count, q_count;
};
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
// Row of line `line` (of `lines`) of an operand, or kNoRow, in two steps: what the
// index says, and what it means, so that a row can be asked for ahead of its use.
// (The index has an entry at least.)
__device__ __forceinline__ uint32_t ask_row(const uint32_t* index, uint32_t line, uint32_t lines) { return index ? index[min(line, max(lines, 1u) - 1u)] : line; }
__device__ __forceinline__ uint32_t judge_row(uint32_t row, uint32_t count, uint32_t line, uint32_t lines) { return line < lines && row < count ? row : kNoRow; }
__device__ __forceinline__ uint32_t gathered_row(const uint32_t* index, uint32_t count, uint32_t line, uint32_t lines) { return judge_row(ask_row(index, line, lines), count, line, lines); }

// Where a workgroup's tile lies: its first outputs, its k, and what P's rows and k
// are counted from (a group's weights in the array of all groups').
struct Place {
    uint32_t p0, q0, k0, k_end, p_line, p_k;
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

// Stager for lines in another order.  Their rows are known before their values
// are asked for: those of rows from the start, those of k (kT) a tile ahead.
template <typename T, uint32_t kB, bool kT, uint32_t kThreads>
struct GatherStager {
    static constexpr uint32_t kChunks = kT ? kB / 8u : 8u;
    static constexpr uint32_t kLoads  = kB * 8u / kThreads;
    Eight<true> held[kLoads];
    uint32_t rows[kLoads], next[kT ? kLoads : 1u];

    static __device__ __forceinline__ uint32_t line(uint32_t i) { return (i * kThreads + threadIdx.x) / kChunks; }
    static __device__ __forceinline__ uint32_t chunk(uint32_t i) { return (i * kThreads + threadIdx.x) % kChunks; }
    __device__ __forceinline__ void begin(const uint32_t* index, uint32_t count, uint32_t first, uint32_t end) {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            if constexpr (kT) next[i] = ask_row(index, first + line(i), end);
            else rows[i] = gathered_row(index, count, first + line(i), end);
        }
    }
    __device__ __forceinline__ Edge place(uint32_t i, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) const {
        return kT ? edge(ld, rows[i], kNoRow, row0 + 8u * chunk(i), n) : edge(ld, rows[i], kNoRow, k0 + 8u * chunk(i), k_end);
    }
    __device__ __forceinline__ void fetch(const T* __restrict__ src, const uint32_t* index, uint32_t count, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) {
        if constexpr (kT) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) rows[i] = judge_row(next[i], count, k0 + line(i), k_end);
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) held[i].fetch(src + place(i, ld, n, row0, k0, k_end).at);
        if constexpr (kT) begin(index, count, k0 + kBK, k_end);
    }
    __device__ __forceinline__ void keep(uint4* lds, const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) const {
        const uint32_t first = value_number(src);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const Edge e                                 = place(i, ld, n, row0, k0, k_end);
            lds[chunk_slot<kB, kT>(line(i), chunk(i))] = settled(held[i].value(first + (uint32_t)e.at), e.down, e.some);
        }
    }
};

// Loader for lines in another order, of an array of less than 2^31 bytes: offsets
// are counted from the array's start.
template <typename T, uint32_t kB, bool kT, uint32_t kThreads>
struct GatherLoader {
    static constexpr uint32_t kChunks = kT ? kB / 8u : 8u;
    static constexpr uint32_t kLoads  = kB * 8u / kThreads;
    const T* base;
    uint32_t offset[kLoads];  // bytes, kBeyond for lines outside; kT: what the index says of the next tile's
    uint32_t k, k_last;       // kT: the next tile's first k, and the end

    static __device__ __forceinline__ uint32_t line(uint32_t i) { return (i * kThreads + threadIdx.x) / kChunks; }
    static __device__ __forceinline__ uint32_t chunk(uint32_t i) { return ((i * kThreads + threadIdx.x) % kChunks) ^ chunk_key<kB, kT>(line(i)); }
    __device__ __forceinline__ void begin(const T* src, const uint32_t* index, uint32_t count, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, uint32_t k_end) {
        base   = src + (kT ? row0 : k0);
        k      = k0;
        k_last = k_end;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            if constexpr (kT) {
                offset[i] = ask_row(index, k + line(i), k_last);
            } else {
                const uint32_t row = gathered_row(index, count, row0 + line(i), n);
                offset[i]          = row != kNoRow ? (row * (uint32_t)ld + 8u * chunk(i)) * 2u : kBeyond;
            }
        }
    }
    __device__ __forceinline__ void issue(uint4* lds, int left, const uint32_t* index, uint32_t count, uint64_t ld, uint32_t n, uint32_t row0) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)0x7FFFFFFF, 0x00020000);
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            uint32_t at = offset[i];
            if constexpr (kT) {
                const uint32_t row = judge_row(offset[i], count, k + line(i), k_last);
                at                 = row != kNoRow && row0 + 8u * chunk(i) < n ? (row * (uint32_t)ld + 8u * chunk(i)) * 2u : kBeyond;
            } else if (left < (int)kBK && (int)(8u * chunk(i)) >= left) {
                at = kBeyond;
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + i * kThreads + wave * 64u), 16, (int)at, 0, 0, 0);
        }
        if constexpr (kT) {
            k += kBK;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) offset[i] = ask_row(index, k + line(i), k_last);
        } else {
            base += kBK;
        }
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

// What the kernels that stream rows begin with: the workgroup's kBP rows of P from p0, 64 k
// at a time, through LDS (kBP * 8 chunks) into the registers of the waves, each of which
// holds 16 kFP of them from wp on for all k; their biases into LDS.
template <typename T, uint32_t kBP, bool kPT, uint32_t kKS, uint32_t kFP, typename Ops, typename Out>
__device__ __forceinline__ void hold_weights(const Ops& A, const Out& out, uint32_t p0, uint32_t wp, uint4* lds, floatx4* lds_bias, typename Vec<T>::x8 (&fp)[kKS][kFP]) {
    const float bias = thread_bias<kBP>(out, p0);
    Stager<T, kBP, kPT, kStreamWaves * 64u, true> stager;
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
// kGather: lines in another order (Ops = GatheredOperands).  more.begin() gives what the
// sums begin with, while the first tiles are on their way.
enum Mode : uint32_t { kDirect, kByChunks, kByWords };
struct NothingMore {
    static constexpr bool kOn = false;
    template <uint32_t kFP, uint32_t kFQ>
    __device__ __forceinline__ uint32_t ask(uint32_t) const { return 0u; }
    __device__ __forceinline__ void ask_more(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) const {}
    template <uint32_t kFP, uint32_t kFQ>
    __device__ __forceinline__ void add(floatx4 (&)[kFP][kFQ], uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) const {}
};
template <typename T, uint32_t kBP, uint32_t kBQ, uint32_t kWP, uint32_t kWQ, uint32_t kDepth, bool kPT, bool kQT, Mode kMode, bool kGather = false, typename Ops, typename Out, typename More = NothingMore>
__device__ __forceinline__ void product(const Ops& A, Out out, const Place& at, const More& more = {}) {
    constexpr uint32_t kThreads = kWP * kWQ * 64u;
    constexpr uint32_t kFP = kBP / kWP / 16u, kFQ = kBQ / kWQ / 16u;
    // Variables of their own, so that the compiler sees that a read of one is no
    // read of what is on its way into another.
    constexpr bool kAligned  = kMode == kDirect;
    constexpr uint32_t kTile = (kBP + kBQ) * 8u;
    static_assert(!kAligned || kDepth == 2u || (kDepth == 4u && !(kGather && kQT)));  // rows of k are loads too
    __shared__ uint4 lds0[kTile], lds1[kAligned ? kTile : 1u], lds2[kAligned && kDepth == 4u ? kTile : 1u], lds3[kAligned && kDepth == 4u ? kTile : 1u];
    __shared__ floatx4 lds_bias[Out::kBias ? kBP / 4u : 1u];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t wp = (wave % kWP) * (kBP / kWP), wq = (wave / kWP) * (kBQ / kWQ);
    const uint32_t p0 = at.p0, q0 = at.q0, k0 = at.k0, k_end = at.k_end;
    const uint32_t p_row = at.p_line + p0, p_rows = at.p_line + A.np;

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
    if constexpr (kSums) take_sums = out.row_sums && p0 == 0u;
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
        // Rows of P in another order: only where k are (dW).
        constexpr bool kGatherP = kGather && kQT;
        std::conditional_t<kGatherP, GatherLoader<T, kBP, kPT, kThreads>, Loader<T, kBP, kPT, kThreads>> load_p;
        std::conditional_t<kGather, GatherLoader<T, kBQ, kQT, kThreads>, Loader<T, kBQ, kQT, kThreads>> load_q;
        if constexpr (kGatherP) load_p.begin((const T*)A.p, A.p_index, A.p_count, A.ldp, A.np, p0, k0, k_end);
        else load_p.begin((const T*)A.p, A.ldp, p_rows, p_row, k0 + at.p_k);
        if constexpr (kGather) load_q.begin((const T*)A.q, A.q_index, A.q_count, A.ldq, A.nq, q0, k0, k_end);
        else load_q.begin((const T*)A.q, A.ldq, A.nq, q0, k0);
        constexpr uint32_t kLoads = kBP * 8u / kThreads + kBQ * 8u / kThreads;
        auto issue = [&](uint4* lds, int left) {
            if constexpr (kGatherP) load_p.issue(lds, left, A.p_index, A.p_count, A.ldp, A.np, p0);
            else load_p.issue(lds, left);
            if constexpr (kGather) load_q.issue(lds + kBP * 8u, left, A.q_index, A.q_count, A.ldq, A.nq, q0);
            else load_q.issue(lds + kBP * 8u, left);
        };
        auto before = [&] {
            keep_bias();
            if constexpr (More::kOn) more.template begin<kFP, kFQ>(acc, p0 + wp, q0 + wq);
        };
        constexpr int kStep = (int)kBK;
        int left            = (int)(k_end - k0);
        if constexpr (kDepth == 2u) {
            // Two tiles a turn; a last odd tile is followed by one of zeros (a way out
            // between the two would keep a second copy of the sums alive).  arrived():
            // everyone's part of the tile has come, and everyone is done with the
            // other buffer.
            issue(lds0, left);
            before();
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
            before();
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
        constexpr bool kGatherP = kGather && kQT;
        static_assert(!kGather || (kMode == kByWords && kDepth == 2u));
        std::conditional_t<kGatherP, GatherStager<T, kBP, kPT, kThreads>, Stager<T, kBP, kPT, kThreads, kMode == kByWords>> stage_p[kDepth - 1u];
        std::conditional_t<kGather, GatherStager<T, kBQ, kQT, kThreads>, Stager<T, kBQ, kQT, kThreads, kMode == kByWords>> stage_q[kDepth - 1u];
        if constexpr (kGatherP) stage_p[0].begin(A.p_index, A.p_count, k0, k_end);
        if constexpr (kGather) stage_q[0].begin(A.q_index, A.q_count, kQT ? k0 : q0, kQT ? k_end : A.nq);
        auto fetch = [&](uint32_t d, uint32_t k) {
            if constexpr (kGatherP) stage_p[d].fetch((const T*)A.p, A.p_index, A.p_count, A.ldp, A.np, p0, k, k_end);
            else stage_p[d].fetch((const T*)A.p, A.ldp, p_rows, p_row, k + at.p_k, k_end + at.p_k);
            if constexpr (kGather) stage_q[d].fetch((const T*)A.q, A.q_index, A.q_count, A.ldq, A.nq, q0, k, k_end);
            else stage_q[d].fetch((const T*)A.q, A.ldq, A.nq, q0, k, k_end);
        };
#pragma unroll
        for (uint32_t d = 0; d < kDepth - 1u; ++d)
            if (k0 + kBK * d < k_end) fetch(d, k0 + kBK * d);
        keep_bias();
        if constexpr (More::kOn) more.template begin<kFP, kFQ>(acc, p0 + wp, q0 + wq);
        for (uint32_t k = k0; k < k_end; k += kBK * (kDepth - 1u)) {
#pragma unroll
            for (uint32_t d = 0; d < kDepth - 1u; ++d) {
                const uint32_t kd = k + kBK * d;
                if (kd < k_end) {
                    if constexpr (kGatherP) stage_p[d].keep(lds0, (const T*)A.p, A.ldp, A.np, p0, kd, k_end);
                    else stage_p[d].keep(lds0, (const T*)A.p, A.ldp, p_rows, p_row, kd + at.p_k, k_end + at.p_k);
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
        if (take_sums && lane < 16u) {  // every p of the product with ones holds the sum
#pragma unroll
            for (uint32_t j = 0; j < kSumsQ; ++j) {
                const uint32_t q = q0 + wq + 16u * (wave % kWP * kSumsQ + j) + lane;
                if (q < out.nq) out.row_sums[q] = sums[j][0];
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

// --------------------------------------------------------------- few tiles
// Products of too few outputs to occupy the card by tiles: what counts is the
// time of one workgroup and the number of launches.  A workgroup has a tile of
// 16 kFP x 16 kFQ outputs, its eight waves every eighth 32 k each; a wave fetches
// its operands from memory itself, several steps at a time and without waiting
// for the others, and the eight sums are added in LDS in their order.  (A
// launch costs the host 3.5 us, about what such a kernel takes; one with 64 x 64
// tiles whose k were split over workgroups and a second one to join them took
// 12 us for 7 x 1601 -> 999, this one 7; backward 37 x 788 -> 64 4 us, in three
// launches 10.)
constexpr uint32_t kFewWaves = 8u, kFewMaxK = 4096u;

// 16 kF rows x 32 k of an operand, any alignment, on its way to one wave; the
// edges as Stager has them.  Rows outside are other rows: their products are in
// outputs that nothing reads.
// kGather: rows in another order, the lane's in `rows`.  kWhole: no edges (whole steps
// of k, and of rows where those are contiguous), and none of their code, which a
// kernel that runs through its own once waits for: 32 rows of 32 adapters, 4096 ->
// 4096, 21 us with it.
template <typename T, uint32_t kF, bool kT, bool kWords, bool kGather = false, bool kWhole = false>
struct FewOperand {
    static_assert(!kGather || !kT);
    using x8 = typename Vec<T>::x8;
    static constexpr uint32_t kChunks = 2u * kF;  // of a line of 16 kF rows (kT)
    Eight<kWords> held[kF];
    uint32_t rows[kGather ? kF : 1u];

    __device__ __forceinline__ uint64_t own(uint32_t i, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0) const {
        const uint32_t lane = threadIdx.x & 63u;
        if constexpr (kGather) return (uint64_t)(rows[i] == kNoRow ? 0u : rows[i]) * ld + k0 + 8u * (lane >> 4);
        if (kT) return (uint64_t)(k0 + (i * 64u + lane) / kChunks) * ld + row0 + 8u * ((i * 64u + lane) % kChunks);
        return (uint64_t)min(row0 + 16u * i + (lane & 15u), n - 1u) * ld + k0 + 8u * (lane >> 4);
    }
    __device__ __forceinline__ Edge place(uint32_t i, uint64_t ld, uint32_t n, uint32_t nk, uint32_t row0, uint32_t k0) const {
        const uint32_t lane = threadIdx.x & 63u;
        if constexpr (kGather) return edge(ld, rows[i], kNoRow, k0 + 8u * (lane >> 4), nk);
        if (kT) return edge(ld, k0 + (i * 64u + lane) / kChunks, nk, row0 + 8u * ((i * 64u + lane) % kChunks), n);
        return edge(ld, min(row0 + 16u * i + (lane & 15u), n - 1u), n, k0 + 8u * (lane >> 4), nk);
    }
    static __device__ __forceinline__ bool inner(uint32_t n, uint32_t nk, uint32_t row0, uint32_t k0) { return kWhole || (k0 + 32u <= nk && (!kT || row0 + 16u * kF <= n)); }

    __device__ __forceinline__ void fetch(uint32_t nk, const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0) {
        uint64_t at[kF];
#pragma unroll
        for (uint32_t i = 0; i < kF; ++i) at[i] = own(i, ld, n, row0, k0);
        if (!inner(n, nk, row0, k0)) {
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) at[i] = place(i, ld, n, nk, row0, k0).at;
        }
#pragma unroll
        for (uint32_t i = 0; i < kF; ++i) held[i].fetch(src + at[i]);
    }
    // The fragments of what was fetched; lds: 1024 kF bytes of the wave's own (kT).
    __device__ __forceinline__ void take(uint32_t nk, const T* __restrict__ src, uint64_t ld, uint32_t n, uint32_t row0, uint32_t k0, char* lds, x8 out[kF]) {
        const uint32_t first = value_number(src);
        uint4 v[kF];
        if (inner(n, nk, row0, k0)) {
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) {
                v[i] = held[i].value(first + (uint32_t)own(i, ld, n, row0, k0));
                if (kGather && rows[i] == kNoRow) v[i] = uint4{0u, 0u, 0u, 0u};
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kF; ++i) {
                const Edge e = place(i, ld, n, nk, row0, k0);
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

constexpr uint32_t few_lds(uint32_t fp, uint32_t fq) { return kFewWaves * std::max(16u * fp * 16u * fq * 4u, 1024u * (fp + fq)); }

template <typename T, uint32_t kFP, uint32_t kFQ, bool kPT, bool kQT, bool kWords, bool kGather = false, bool kWhole = false, typename Ops, typename Out, typename More = NothingMore>
__device__ __forceinline__ void few_tile(const Ops& A, Out out, const Place& at, char* lds, float* lds_sums, uint32_t* lds_rows = nullptr, const More& more = {}) {
    const uint32_t p0 = at.p0, q0 = at.q0;
    constexpr bool kSums = std::is_same_v<Out, SumOut>;
    constexpr uint32_t kDepth = kFP * kFQ <= 2u ? 8u : kFP * kFQ == 4u ? 3u : 2u;  // steps on their way
    constexpr uint32_t kSP = 16u * kFP, kEights = 16u * kFQ * kSP / 8u;
    using x8 = typename Vec<T>::x8;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;

    // What the outputs need besides the sums: the thread's eight outputs.
    const uint32_t row = threadIdx.x / (kSP / 8u), col = 8u * (threadIdx.x % (kSP / 8u)), p = p0 + col;
    const uint32_t n = threadIdx.x < kEights && q0 + row < out.nq && p < out.np ? min(8u, out.np - p) : 0u;
    floatx8 bias = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    typename Out::Aux aux;
    auto ask_outputs = [&] {
        if constexpr (Out::kBias) {
            if (out.bias) {
#pragma unroll
                for (uint32_t r = 0; r < 8u; ++r) bias[r] = r < n ? out.bias[p + r] : 0.0f;
            }
        }
        aux = out.load(q0, row, p, n);
    };
    if constexpr (!kGather) ask_outputs();

    floatx4 acc[kFP][kFQ], sums[kFQ];
#pragma unroll
    for (uint32_t j = 0; j < kFQ; ++j) {
        sums[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t i = 0; i < kFP; ++i) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const bool take_sums = kSums && p0 == 0u;
    x8 ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = (T)1.0f;
    FewOperand<T, kFP, kPT, kWords, false, kWhole> op[kDepth];
    FewOperand<T, kFQ, kQT, kWords, kGather, kWhole> oq[kDepth];
    char* mine = lds + wave * 1024u * (kFP + kFQ);
    auto fetch = [&](uint32_t d, uint32_t k) {
        op[d].fetch(A.nk + at.p_k, (const T*)A.p, A.ldp, at.p_line + A.np, at.p_line + p0, k + at.p_k);
        oq[d].fetch(A.nk, (const T*)A.q, A.ldq, A.nq, q0, k);
    };
    constexpr uint32_t kStride = 32u * kFewWaves;
    auto ask_steps = [&](auto one) {
#pragma unroll
        for (uint32_t d = 0; d < kDepth; ++d)
            if (32u * wave + kStride * d < A.nk) one(d, 32u * wave + kStride * d);
    };
    // Loads come back in their order, so what addresses are made of is asked for
    // first, then what needs no address from memory, and then the rest; what else
    // belongs to the sums is added last.
    auto asked = more.template ask<kFP, kFQ>(q0);
    if constexpr (kGather) {
        uint32_t rows[kFQ];
#pragma unroll
        for (uint32_t j = 0; j < kFQ; ++j) rows[j] = ask_row(A.q_index, q0 + 16u * j + (lane & 15u), A.nq);
        ask_steps([&](uint32_t d, uint32_t k) { op[d].fetch(A.nk + at.p_k, (const T*)A.p, A.ldp, at.p_line + A.np, at.p_line + p0, k + at.p_k); });
#pragma unroll
        for (uint32_t j = 0; j < kFQ; ++j)
#pragma unroll
            for (uint32_t d = 0; d < kDepth; ++d) oq[d].rows[j] = judge_row(rows[j], A.q_count, q0 + 16u * j + (lane & 15u), A.nq);
        ask_steps([&](uint32_t d, uint32_t k) { oq[d].fetch(A.nk, (const T*)A.q, A.ldq, A.nq, q0, k); });
        more.ask_more(asked, p0, q0, wave, kFewWaves);
        find_rows<16u * kFQ>(out, lds_rows, q0, out.nq);
        __syncthreads();
        ask_outputs();
    } else {
        ask_steps(fetch);
    }
    for (uint32_t k = 32u * wave; k < A.nk; k += kStride * kDepth) {
#pragma unroll
        for (uint32_t d = 0; d < kDepth; ++d) {
            const uint32_t kd = k + kStride * d;
            if (kd < A.nk) {
                x8 fp[kFP], fq[kFQ];
                op[d].take(A.nk + at.p_k, (const T*)A.p, A.ldp, at.p_line + A.np, at.p_line + p0, kd + at.p_k, mine, fp);
                oq[d].take(A.nk, (const T*)A.q, A.ldq, A.nq, q0, kd, mine + 1024u * kFP, fq);
                if (kd + kStride * kDepth < A.nk) fetch(d, kd + kStride * kDepth);
#pragma unroll
                for (uint32_t i = 0; i < kFP; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < kFQ; ++j) acc[i][j] = Vec<T>::mfma(fp[i], fq[j], acc[i][j]);
                if (take_sums) {
#pragma unroll
                    for (uint32_t j = 0; j < kFQ; ++j) sums[j] = Vec<T>::mfma(ones, fq[j], sums[j]);
                }
            }
        }
    }

    more.add(acc, asked, p0, q0, wave, kFewWaves);
    __syncthreads();  // the waves' own pieces become those of the sums
    floatx4* strips = reinterpret_cast<floatx4*>(lds);
    constexpr uint32_t kStrip = 16u * kFQ * kSP / 4u;
#pragma unroll
    for (uint32_t j = 0; j < kFQ; ++j) {
        const uint32_t r = 16u * j + (lane & 15u);
#pragma unroll
        for (uint32_t i = 0; i < kFP; ++i) strips[wave * kStrip + r * (kSP / 4u) + ((4u * i + (lane >> 4)) ^ (r & 3u))] = acc[i][j];
        if (take_sums && lane < 16u) lds_sums[wave * 16u * kFQ + r] = sums[j][0];
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
        if (take_sums && out.row_sums && threadIdx.x < 16u * kFQ && q0 + threadIdx.x < out.nq) {
            float v = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kFewWaves; ++w) v += lds_sums[w * 16u * kFQ + threadIdx.x];
            out.row_sums[q0 + threadIdx.x] = v;
        }
    }
}

// ------------------------------------------------------------------- host
constexpr uint32_t kMaxFeatures = 1u << 16, kMaxStride = 1u << 20, kMaxRows = 1u << 30;

inline bool aligned(const void* p, uint64_t bytes) { return ((uintptr_t)p & (bytes - 1u)) == 0u; }
inline uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1u) / b); }

struct Workspace {
    float* data;
    uint64_t bytes;
};

// Whether an operand's rows may start at odd values.
inline bool odd_rows(const void* p, uint64_t ld) { return (((uintptr_t)p >> 1 | ld) & 1u) != 0u; }
// Whether an operand's chunks of 8 along its contiguous length are whole and aligned.
inline bool whole_chunks(const void* p, uint64_t ld, uint32_t contiguous) { return aligned(p, 16u) && ld % 8u == 0u && contiguous % 8u == 0u; }

// A layer's descriptor with its defaults filled in, or what is wrong with it.
NerfStatus check_desc(const NerfExtLinearDesc* desc, NerfExtLinearDesc& d, const char* fn);

}  // namespace linear
}  // namespace nerf_hip
