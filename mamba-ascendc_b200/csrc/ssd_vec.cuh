// Element types of the operators that take more than fp32 (short convolution, selective scan, norm) and their loads and
// stores: a thread owns V consecutive elements and holds them in fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ssd_host.h"

namespace ssd {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void pair_from_f(__nv_bfloat16* p, float a, float b) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void pair_from_f(__half* p, float a, float b) {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b);
}

// The plain vector of BYTES bytes.
template <int BYTES>
struct Bits;
template <>
struct Bits<2> { using type = unsigned short; };
template <>
struct Bits<4> { using type = unsigned int; };
template <>
struct Bits<8> { using type = uint2; };
template <>
struct Bits<16> { using type = uint4; };

// V elements as they lie in memory; V * sizeof(T) is 2, 4, 8, 16 or a multiple of 16.
template <class T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
    T v[V];
};

// V elements from p, n of them in range (the rest zero), not yet converted: a load that is to be in flight under other work
// must not be followed by its conversion, at which the warp would wait.  VECTOR: p is aligned for the whole vector and n is
// 0 or V.  KEPT: the memory is written by this kernel as well; otherwise the read may pass stores.
template <bool VECTOR, bool KEPT, int V, class T>
__device__ __forceinline__ void load_raw(Pack<T, V>& raw, const T* p, int n) {
    constexpr int kStep = VECTOR ? (sizeof(raw) < 16 ? sizeof(raw) : 16) : sizeof(T), kLoads = sizeof(raw) / kStep;
    using B = typename Bits<kStep>::type;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        B v{};
        if (VECTOR ? n > 0 : i < n) v = KEPT ? reinterpret_cast<const B*>(p)[i] : __ldg(reinterpret_cast<const B*>(p) + i);
        reinterpret_cast<B*>(&raw)[i] = v;
    }
}
template <int V, class T>
__device__ __forceinline__ void unpack(float (&f)[V], const Pack<T, V>& raw) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f(raw.v[i]);
}
// The same into shared memory without waiting, zeros if not `in`; a thread waits for its own copies.
template <int V, class T>
__device__ __forceinline__ void copy_async(Pack<T, V>& to, const T* p, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(&to))), "l"(p),
                 "n"(sizeof(to)), "r"(in ? static_cast<int>(sizeof(to)) : 0)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
template <bool VECTOR, int V, class T>
__device__ __forceinline__ void load_f(float (&f)[V], const T* p, int n) {
    Pack<T, V> raw;
    load_raw<VECTOR, false>(raw, p, n);
    unpack(f, raw);
}
// of memory that this kernel writes as well
template <bool VECTOR, int V, class T>
__device__ __forceinline__ void load_kept(float (&f)[V], const T* p, int n) {
    Pack<T, V> raw;
    load_raw<VECTOR, true>(raw, p, n);
    unpack(f, raw);
}
template <bool VECTOR, int V, class T>
__device__ __forceinline__ void store_raw(T* p, const Pack<T, V>& raw, int n) {
    constexpr int kStep = VECTOR ? (sizeof(raw) < 16 ? sizeof(raw) : 16) : sizeof(T), kStores = sizeof(raw) / kStep;
    using B = typename Bits<kStep>::type;
#pragma unroll
    for (int i = 0; i < kStores; ++i)
        if (VECTOR ? n > 0 : i < n) reinterpret_cast<B*>(p)[i] = reinterpret_cast<const B*>(&raw)[i];
}
template <bool VECTOR, int V, class T>
__device__ __forceinline__ void store_f(T* p, const float (&f)[V], int n) {
    Pack<T, V> raw;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {  // two values a conversion
#pragma unroll
        for (int i = 0; i < V; i += 2) pair_from_f(raw.v + i, f[i], f[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) raw.v[i] = from_f<T>(f[i]);
    }
    store_raw<VECTOR>(p, raw, n);
}

// Parameters come in fp32 or in the activations' type, by a flag that is the same for every thread.
template <class T>
__device__ __forceinline__ float load_param(const void* p, int f32, long long i) {
    return f32 ? static_cast<const float*>(p)[i] : to_f(static_cast<const T*>(p)[i]);
}
template <class T>
__device__ __forceinline__ void store_param(void* p, int f32, long long i, float v) {
    if (f32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<T*>(p)[i] = from_f<T>(v);
}

__device__ __forceinline__ float ex2f(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float rcpf(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// 1 / (1 + e^-v): exact limits at both ends (e^-v overflows to infinity, whose reciprocal is 0)
__device__ __forceinline__ float sigmoid_fast(float v) { return rcpf(1.f + ex2f(-v * kLog2e)); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// ---- sequences: a batch [rows, tokens], or packed one behind another as `cu` [rows + 1] says, cut into items of `span`
// tokens so that an item lies in one sequence.  Sequence s has ceil(length / span) items, one if it is empty; packed, item
// numbers start at start_s / span + s, which leaves room for them whatever the lengths, and numbers in between are idle.
// Tokens behind the last packed sequence are one more sequence, `pad`, whose outputs are zeros.
struct SeqMap {
    const int* cu;
    long long tokens;  // of a batch row, or all packed ones
    int rows, span;
    __host__ __device__ long long per_row() const { return tokens > span ? (tokens + span - 1) / span : 1; }
    __host__ __device__ long long items() const { return cu == nullptr ? per_row() * rows : tokens / span + rows + 1; }
    // start of sequence s; whatever `cu` holds, nothing lies outside the tokens
    __device__ long long start(int s) const {
        if (s == 0) return 0;
        const long long v = cu[s];
        return v < 0 ? 0 : v > tokens ? tokens : v;
    }
};
struct Span {
    int seq, seg;
    bool pad, first, last;
    long long origin;  // packed: first token of the sequence; batch: 0
    int len, t0, t1;   // tokens of the sequence, and of this item
};
// Called by all threads of the CTA; false for an idle item.
__device__ __forceinline__ bool locate(const SeqMap& m, long long item, Span& s) {
    if (m.cu == nullptr) {
        const long long per = m.per_row();
        s.seq = static_cast<int>(item / per);
        s.seg = static_cast<int>(item - s.seq * per);
        s.origin = 0;
        s.len = static_cast<int>(m.tokens);
        s.pad = false;
    } else {
        int below = 0;  // sequences (the padding included) whose items start at or before this one
        for (int base = 0; base <= m.rows; base += blockDim.x) {
            const int q = base + threadIdx.x;
            below += __syncthreads_count(q <= m.rows && m.start(q) / m.span + q <= item);
        }
        s.seq = max(below - 1, 0);
        s.pad = s.seq == m.rows;
        s.origin = m.start(s.seq);
        const long long end = s.pad ? m.tokens : m.start(s.seq + 1);
        s.len = static_cast<int>(max(end - s.origin, 0LL));
        const long long seg = item - (s.origin / m.span + s.seq);
        if (seg < 0 || (seg > 0 && seg * m.span >= s.len)) return false;
        s.seg = static_cast<int>(seg);
    }
    s.t0 = s.seg * m.span;
    s.t1 = min(s.len - s.t0, m.span) + s.t0;
    s.first = s.seg == 0;
    s.last = s.t1 == s.len;
    return true;
}
// Row of token t: the distance in elements from the tensor's start.
__device__ __forceinline__ long long token_row(const SeqMap& m, const Span& s, long long batch_stride, long long token_stride,
                                               int t) {
    return (m.cu == nullptr ? s.seq * batch_stride : 0) + (s.origin + t) * token_stride;
}

// Rows at a distance that fits 31 bits in bytes (the entry points refuse others), so that a row's address is one multiply-add.
template <class T>
struct Rows {
    const char* base;
    int step;
    __device__ __forceinline__ Rows(const T* first, int64_t elements)
        : base(reinterpret_cast<const char*>(first)), step(static_cast<int>(elements) * static_cast<int>(sizeof(T))) {}
    __device__ __forceinline__ const T* at(int t) const {
        return reinterpret_cast<const T*>(base + static_cast<long long>(t) * step);
    }
    __device__ __forceinline__ T* to(int t) const { return const_cast<T*>(at(t)); }
};
template <class... S>
inline bool row_steps(S... elements) {
    return ((elements >= 0 && elements < (1 << 29)) && ...);
}

// ---- rows of a generation step that name the same slot.  Of a CTA's ROWS rows from row0 on: bit i, row i's slot is taken by an
// earlier row; bit 16 + i, a later row names it too.  Every warp leaves what its threads found in flags[warp]; any_flag
// joins them behind a barrier of the caller's.
template <int ROWS, int THREADS>
__device__ __forceinline__ void shared_slots(const int (&slot)[ROWS], const int* slots, int rows, int row0, unsigned* flags) {
    if (slots == nullptr) return;
    unsigned bits = 0;
    for (int r = threadIdx.x; r < rows; r += THREADS) {
        const int other = __ldg(slots + r);
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            if (other == slot[i] && r != row0 + i) bits |= r < row0 + i ? 1u << i : 0x10000u << i;
    }
    bits = __reduce_or_sync(0xffffffffu, bits);
    if ((threadIdx.x & 31) == 0) flags[threadIdx.x >> 5] = bits;
}
template <int WARPS>
__device__ __forceinline__ unsigned any_flag(const unsigned (&flags)[WARPS]) {
    unsigned bits = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) bits |= flags[w];
    return bits;
}

// ---- sums over the rows of a table [rows][cols] in a fixed order: the second half of gradients of parameters.
// Cell (r, c) of `out` gets the sum of column `col`; StoreCol(col, sum) writes it.
constexpr int kSumCols = 32, kSumRows = 32;
template <class StoreCol>
__device__ __forceinline__ void column_sums(const float* table, long long rows, long long cols, StoreCol store) {
    __shared__ float part[kSumRows][kSumCols];
    const long long c = static_cast<long long>(blockIdx.x) * kSumCols + threadIdx.x % kSumCols;
    const int r0 = threadIdx.x / kSumCols;
    float sum = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (long long r = r0; r < rows; r += kSumRows) sum += table[r * cols + c];
    }
    part[r0][threadIdx.x % kSumCols] = sum;
    __syncthreads();
    if (r0 == 0 && c < cols) {
        for (int r = 1; r < kSumRows; ++r) sum += part[r][threadIdx.x];
        store(c, sum);
    }
}

// `f` with the element type that `dtype` names.
template <class F>
int with_type(int dtype, F f) {
    switch (dtype) {
        case SSD_F32: return f(float{});
        case SSD_BF16: return f(__nv_bfloat16{});
        case SSD_F16: return f(__half{});
        default: return SSD_ERR_UNSUPPORTED;
    }
}
inline bool multiple_of(long long v, long long m) { return v % m == 0; }
template <class... P>
inline bool aligned_to(size_t bytes, const P*... p) {
    return ((reinterpret_cast<uintptr_t>(p) | ... | uintptr_t{0}) & (bytes - 1)) == 0;
}

}  // namespace ssd
