// Shared by the kernels of the selective scan (ssd_selective_fwd.cu, _bwd.cu, _step.cu).
#pragma once

#include "ssd_vec.cuh"

namespace ssd {

constexpr int kScanMaxState = 128;
constexpr int kScanCheckpoint = 64;  // tokens between the states that backward starts from

// Two fp32 values side by side.  (The packed fp32 instructions take two cycles each, so they save nothing, and tie registers in
// pairs: the forward pass before its staging warps took 559 us with them and 483 without.)
struct alignas(8) F2 {
    float x, y;
};
__device__ __forceinline__ F2 pack2(float lo, float hi) { return {lo, hi}; }
__device__ __forceinline__ float2 unpack2(F2 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { return {fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)}; }
// log(1 + e^v) = max(v, 0) + log1p(e) with e = e^-|v| in [0, 1]; log1p(e) = 2 atanh(s) with s = e / (2 + e) in [0, 1/3], and
// 2 atanh(s) / s is taken as the polynomial in s^2 that meets it at the Chebyshev nodes of [0, 1/9] (off by 8e-9 of the value at most).
// Relative accuracy also where v is very negative.
__device__ __forceinline__ float softplus_series(float v) {
    const float e = ex2f(fabsf(v) * -kLog2e);
    const float s = e * rcpf(2.f + e), q = s * s;
    float p = 0.28157780f;
    p = fmaf(p, q, 0.27965158f);
    p = fmaf(p, q, 0.40024596f);
    p = fmaf(p, q, 0.66666323f);
    p = fmaf(p, q, 2.f);
    return fmaf(p, s, fmaxf(v, 0.f));
}

// A in powers of two.  Minus infinity (a column that keeps nothing) becomes the lowest number that a step of zero, as tokens
// behind the end of a sequence have it, turns into zero and not into NaN.
__device__ __forceinline__ float decay_rate(float a) {
    const float v = a * kLog2e;
    return v == -INFINITY ? -3.0e38f : v;
}

// exp(dt A).  The approximate exponential is low by 5e-9 of its value on average for arguments from -2^-8 to 0 (measured over a
// million in each binade; single values are off by up to 8e-8 either way), and a state that lives for thousands of tokens adds
// that up: 1.5e-5 in gradients of A.  An argument moved up by 8e-9 leaves 8e-10; where arguments are larger the shift is lost
// in their rounding, and there the states are short-lived.  A step of zero still gives 1.
__device__ __forceinline__ float decay(float dt, float rate) { return ex2f(fmaf(dt, rate, 8.0e-9f)); }

// The channels of a CTA lie in one group.
struct ScanBlocks {
    int per_cta, per_group;  // channels of a CTA, CTAs of a group
    __host__ __device__ int count(int groups) const { return per_group * groups; }
};
inline ScanBlocks scan_blocks(int channels, int groups, int per_cta) {
    const int mine = channels / groups;
    return {per_cta, (mine + per_cta - 1) / per_cta};
}
struct ChannelBlock {
    int group, first, n;  // first channel and how many there are
};
__device__ __forceinline__ ChannelBlock channel_block(const ScanBlocks& b, int block, int channels, int groups) {
    const int mine = groups == 1 ? channels : channels / groups, group = groups == 1 ? 0 : block / b.per_group;
    const int at = (block - group * b.per_group) * b.per_cta;
    return {group, group * mine + at, min(mine - at, b.per_cta)};
}

template <class T>
__device__ __forceinline__ float2 pair_f(const Pack<T, 2>& raw) {
    return make_float2(to_f(raw.v[0]), to_f(raw.v[1]));
}
// Two channels of a row; n of them exist.
template <bool VECTOR, class T>
__device__ __forceinline__ float2 load_pair(const T* p, int n) {
    float f[2];
    load_f<VECTOR>(f, p, n);
    return make_float2(f[0], f[1]);
}
template <bool VECTOR, class T>
__device__ __forceinline__ void store_pair(T* p, float2 v, int n) {
    const float f[2] = {v.x, v.y};
    store_f<VECTOR>(p, f, n);
}

// Token 0 of the sequence: the distance in elements from the tensor's start.
__device__ __forceinline__ long long first_row(const SeqMap& m, const Span& s, const int64_t* strides) {
    return m.cu == nullptr ? s.seq * strides[0] : s.origin * strides[1];
}

// Whether two channels and four state columns can be loaded at once.
inline bool scan_pairs(const SsdScanArgs& a, size_t element) {
    const int64_t strides = a.x_strides[0] | a.x_strides[1] | a.dt_strides[0] | a.dt_strides[1] | a.z_strides[0] | a.z_strides[1];
    const int64_t shared = a.b_strides[0] | a.b_strides[1] | a.b_strides[2] | a.c_strides[0] | a.c_strides[1] | a.c_strides[2] | a.dstate;
    return aligned_to(2 * element, a.x, a.dt, a.z, a.out) && (strides & 1) == 0 && a.channels / a.groups % 2 == 0 &&
           aligned_to(4 * element, a.bm, a.cm) && (shared & 3) == 0;
}
inline SeqMap scan_map(const SsdScanArgs& a, int span) { return SeqMap{a.cu_seqlens, a.tokens, a.rows, span}; }
int scan_check(const SsdScanArgs& a);

// ---- long sequences of few channels are cut into segments, whose states are found in two more passes: each segment's own
// contribution from a zero state (in either direction), then a walk over the segments.
// work: [items][dstate][channels] states, then [items][channels] sums of dt.
struct ScanSegments {
    int span;           // tokens of a segment
    long long items;    // of the map
    bool split;         // whether any sequence can have more than one
};
ScanSegments scan_segments(const SsdScanArgs& a, int per_cta, int slots);
inline size_t scan_segment_floats(const SsdScanArgs& a, const ScanSegments& s) {
    return s.split ? static_cast<size_t>(s.items) * a.channels * (a.dstate + 1) : 0;
}
// Leaves in `work` each segment's state before its first token (backward: the gradient of the state behind its last one).
int scan_segment_states(const SsdScanArgs& a, const ScanSegments& s, float* work, const void* dout, const float* dfinal,
                        cudaStream_t stream);

}  // namespace ssd
