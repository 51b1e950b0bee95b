// Selective scan of one token of each sequence: the state out of a cache, moved on by the token, and back.
//
// What bounds it: HBM, the state once in each direction (fp32, 4 dstate bytes per channel each way against 8 of the token).
// Lanes lie along the state (four columns each) and then along the channels, so that a warp reads and writes whole lines;
// a thread takes kRows rows of the batch with the loads of all their states in flight, and keeps A.
#include "ssd_selective.cuh"

namespace ssd {

namespace {

constexpr int kStepThreads = 128;

// LPC lanes hold a channel's columns, four each.  VECTOR: dstate is a multiple of four, and states, B and C
// are aligned for four at once.
template <class T, int LPC, int ROWS, bool VECTOR>
__global__ void __launch_bounds__(kStepThreads)
selective_step_kernel(const SsdScanStepArgs a, int channel_blocks) {
    constexpr int kChannels = kStepThreads / LPC;
    __shared__ unsigned flags;  // bit i: row i's slot is taken by an earlier row; bit 16 + i: a later row names it too
    const int row0 = blockIdx.x / channel_blocks * ROWS;
    const int c = blockIdx.x % channel_blocks * kChannels + threadIdx.x / LPC;
    const int part = threadIdx.x % LPC, n0 = part * 4, nn = max(min(a.dstate - n0, 4), 0);
    const bool live = c < a.channels;
    const int g = live ? c / (a.channels / a.groups) : 0;

    // every load of the rows in flight before the first is used
    long long slot[ROWS];
    Pack<float, 4> hr[ROWS];
    Pack<T, 4> br[ROWS], cr[ROWS];
    Pack<T, 1> xr[ROWS], dr[ROWS], zr[ROWS];
    auto request = [&](Pack<T, 1>& xv, Pack<T, 1>& dv, Pack<T, 1>& zv, Pack<T, 4>& bv, Pack<T, 4>& cv, long long row, bool in) {
        load_raw<true, false>(xv, static_cast<const T*>(a.x) + row * a.x_stride + c, in);
        load_raw<true, false>(dv, static_cast<const T*>(a.dt) + row * a.dt_stride + c, in);
        load_raw<true, false>(zv, static_cast<const T*>(a.z) + row * a.z_stride + c, in && a.z != nullptr);
        load_raw<VECTOR, false>(bv, static_cast<const T*>(a.bm) + row * a.b_strides[0] + g * a.b_strides[1] + n0, in ? nn : 0);
        load_raw<VECTOR, false>(cv, static_cast<const T*>(a.cm) + row * a.c_strides[0] + g * a.c_strides[1] + n0, in ? nn : 0);
    };
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        slot[i] = row >= a.rows ? -1 : a.slots != nullptr ? a.slots[row] : row;
        if (slot[i] >= a.slot_count) slot[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const bool in = live && slot[i] >= 0;
        load_raw<VECTOR, true>(hr[i], a.state + (in ? slot[i] * a.state_stride + static_cast<long long>(c) * a.dstate + n0 : 0),
                               in ? nn : 0);
        request(xr[i], dr[i], zr[i], br[i], cr[i], in ? row0 + i : 0, in);
    }
    float a2[4];
    load_f<VECTOR>(a2, a.A + (live ? static_cast<long long>(c) * a.dstate + n0 : 0), live ? nn : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) a2[j] *= kLog2e;
    const float bias = live && a.dt_bias != nullptr ? a.dt_bias[c] : 0.f, skip = live && a.D != nullptr ? a.D[c] : 0.f;

    unsigned found = 0;
    if (a.slots != nullptr) {
        if (threadIdx.x == 0) flags = 0;
        __syncthreads();
        unsigned bits = 0;
        for (int r = threadIdx.x; r < a.rows; r += kStepThreads) {
            const int other = a.slots[r];
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
                if (other == slot[i] && r != row0 + i) bits |= r < row0 + i ? 1u << i : 0x10000u << i;
        }
        if (bits != 0) atomicOr(&flags, bits);
        __syncthreads();
        found = flags;
    }

    // one token: the state moved on, and its output
    auto token = [&](float (&s)[4], const Pack<T, 1>& xp, const Pack<T, 1>& dp, const Pack<T, 1>& zp, const Pack<T, 4>& bp,
                     const Pack<T, 4>& cp, int row) {
        float b[4], cv[4];
        unpack(b, bp);
        unpack(cv, cp);
        const float xv = to_f(xp.v[0]);
        float d = to_f(dp.v[0]) + bias;
        if (a.softplus) d = softplus_series(d);
        const float u = d * xv;
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = fmaf(ex2f(d * a2[j]), s[j], u * b[j]);
            y = fmaf(cv[j], s[j], y);
        }
#pragma unroll
        for (int o = LPC / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (live && part == 0) {
            y = fmaf(skip, xv, y);
            if (a.z != nullptr) {
                const float zv = to_f(zp.v[0]);
                y *= zv * sigmoid_fast(zv);
            }
            static_cast<T*>(a.out)[static_cast<long long>(row) * a.channels + c] = from_f<T>(y);
        }
    };
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        if (row >= a.rows) break;
        if (slot[i] < 0) {
            if (live && part == 0) static_cast<T*>(a.out)[static_cast<long long>(row) * a.channels + c] = from_f<T>(0.f);
            continue;
        }
        if (found & (1u << i)) continue;  // the first row with this slot takes them all
        float h[4];
        unpack(h, hr[i]);
        token(h, xr[i], dr[i], zr[i], br[i], cr[i], row);
        if (found & (0x10000u << i))
            for (int r = row + 1; r < a.rows; ++r)
                if (a.slots[r] == slot[i]) {
                    Pack<T, 1> xv, dv, zv;
                    Pack<T, 4> bv, cv;
                    request(xv, dv, zv, bv, cv, r, live);
                    token(h, xv, dv, zv, bv, cv, r);
                }
        if (live) store_f<VECTOR>(a.state_out + slot[i] * a.state_out_stride + static_cast<long long>(c) * a.dstate + n0, h, nn);
    }
}

}  // namespace

}  // namespace ssd

extern "C" int ssd_selective_scan_step(const SsdScanStepArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdScanStepArgs& a = *args;
    if (a.rows <= 0 || a.channels <= 0 || a.dstate <= 0 || a.groups <= 0 || a.channels % a.groups != 0 || a.slot_count <= 0 ||
        (a.slots == nullptr && a.slot_count < a.rows))
        return SSD_ERR_SHAPE;
    if (a.dstate > kScanMaxState) return SSD_ERR_UNSUPPORTED;
    if (!a.x || !a.dt || !a.A || !a.bm || !a.cm || !a.state || !a.state_out || !a.out) return SSD_ERR_NULL;
    const bool vector = a.dstate % 4 == 0 && aligned16(a.A, a.state, a.state_out) && multiple_of(a.state_stride, 4) &&
                        multiple_of(a.state_out_stride, 4) && multiple_of(a.b_strides[0] | a.b_strides[1], 4) &&
                        multiple_of(a.c_strides[0] | a.c_strides[1], 4) &&
                        aligned_to(a.dtype == SSD_F32 ? 16 : 8, a.bm, a.cm);
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const auto launch = [&](auto lpc, auto rows) {
            constexpr int LPC = decltype(lpc)::value, ROWS = decltype(rows)::value;
            const int channel_blocks = (a.channels + kStepThreads / LPC - 1) / (kStepThreads / LPC);
            const long long blocks = static_cast<long long>((a.rows + ROWS - 1) / ROWS) * channel_blocks;
            if (blocks > 0x7fffffffLL) return static_cast<int>(SSD_ERR_RANGE);
            launch_plain(vector ? selective_step_kernel<T, LPC, ROWS, true> : selective_step_kernel<T, LPC, ROWS, false>,
                         static_cast<unsigned>(blocks), kStepThreads, 0, reinterpret_cast<cudaStream_t>(stream), a, channel_blocks);
            return launch_status();
        };
        const auto with_rows = [&](auto lpc) {
            // several rows of a thread share A; one where that would leave SMs without a CTA
            constexpr int LPC = decltype(lpc)::value;
            const long long ctas = static_cast<long long>(a.rows) * ((a.channels + kStepThreads / LPC - 1) / (kStepThreads / LPC));
            return ctas >= 16LL * sm_count() ? launch(lpc, std::integral_constant<int, 4>{})
                                             : launch(lpc, std::integral_constant<int, 1>{});
        };
        if (a.dstate <= 16) return with_rows(std::integral_constant<int, 4>{});
        if (a.dstate <= 32) return with_rows(std::integral_constant<int, 8>{});
        if (a.dstate <= 64) return with_rows(std::integral_constant<int, 16>{});
        return with_rows(std::integral_constant<int, 32>{});
    });
}
