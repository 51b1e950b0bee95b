// Selective scan of one token of each sequence: the state out of a cache, moved on by the token, and back.
//
// What bounds it: HBM, the state once in each direction (fp32, 4 dstate bytes per channel each way against 8 of the token),
// as long as little else is done per state column: what belongs to a (row, channel), softplus, gate and skip connection, is
// formed once by one thread and passes to the channel's lanes through shared memory, as do B and C in fp32.  A lane has eight
// columns of a channel (32 bytes, one access), lanes lie along the columns and then along the channels; a thread takes
// ROWS rows of the batch with the loads of all their states in flight, and keeps A.
#include "ssd_selective.cuh"

namespace ssd {

namespace {

constexpr int kStepThreads = 128, kStepCols = 8;

// Eight floats at a 32-byte boundary.
__device__ __forceinline__ void load8(float (&f)[kStepCols], const float* p) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7])
                 : "l"(p));
}
__device__ __forceinline__ void store8(float* p, const float (&f)[kStepCols]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]),
                 "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                 : "memory");
}

// LPC lanes hold a channel's columns.  VECTOR: dstate is a multiple of eight and the states lie at 32-byte boundaries.
template <class T, int LPC, int ROWS, bool VECTOR>
__global__ void __launch_bounds__(kStepThreads)
selective_step_kernel(const SsdScanStepArgs a, const ScanBlocks b) {
    constexpr int kChannels = kStepThreads / LPC, kWide = LPC * kStepCols;  // channels of a CTA, columns with those behind dstate
    __shared__ unsigned flags[kStepThreads / 32];  // see shared_slots
    __shared__ float4 token[ROWS][kChannels];  // dt, dt x, gate, gated skip connection
    __shared__ __align__(16) float shared[ROWS][2][kWide];
    const int row0 = blockIdx.x * ROWS, tid = threadIdx.x;
    const ChannelBlock cb = channel_block(b, blockIdx.y, a.channels, a.groups);
    const int mine = tid / LPC, c = cb.first + mine, part = tid % LPC, n0 = part * kStepCols;
    const int nn = mine < cb.n ? max(min(a.dstate - n0, kStepCols), 0) : 0;
    const long long own = static_cast<long long>(c) * a.dstate + n0;

    int slot[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        slot[i] = row >= a.rows ? -1 : a.slots != nullptr ? a.slots[row] : row;
        if (slot[i] >= a.slot_count) slot[i] = -1;
    }
    float h[ROWS][kStepCols], a2[kStepCols];
    const auto load_state = [&](float (&f)[kStepCols], const float* p, bool in) {
        if constexpr (VECTOR) {
            if (in && nn > 0) {
                load8(f, p);
            } else {
#pragma unroll
                for (int j = 0; j < kStepCols; ++j) f[j] = 0.f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < kStepCols; ++j) f[j] = in && j < nn ? p[j] : 0.f;
        }
    };
#pragma unroll
    for (int i = 0; i < ROWS; ++i) load_state(h[i], a.state + static_cast<long long>(slot[i]) * a.state_stride + own, slot[i] >= 0);

    // what belongs to a token: one thread per (row, channel), and per (row, column) of B and C
    const Rows<T> xs(static_cast<const T*>(a.x) + cb.first, a.x_stride), dts(static_cast<const T*>(a.dt) + cb.first, a.dt_stride);
    const Rows<T> zs(static_cast<const T*>(a.z) + cb.first, a.z_stride);
    const Rows<T> bs(static_cast<const T*>(a.bm) + cb.group * a.b_strides[1], a.b_strides[0]);
    const Rows<T> cs(static_cast<const T*>(a.cm) + cb.group * a.c_strides[1], a.c_strides[0]);
    const auto stage_token = [&](int i, int row, int k) {
        if (k < cb.n) {
            const int ch = cb.first + k;
            const float xv = to_f(__ldg(xs.at(row) + k));
            float d = to_f(__ldg(dts.at(row) + k));
            float gate = 1.f;
            if (a.z != nullptr) {
                const float zv = to_f(__ldg(zs.at(row) + k));
                gate = zv * sigmoid_fast(zv);
            }
            if (a.dt_bias != nullptr) d += a.dt_bias[ch];
            if (a.softplus) d = softplus_series(d);
            const float skip = a.D != nullptr ? a.D[ch] * xv : 0.f;
            token[i][k] = make_float4(d, d * xv, gate, skip);
        }
    };
    const auto stage_shared = [&](int i, int row, int k) {
        const int n = k % kWide;
        shared[i][k / kWide][n] = n < a.dstate ? to_f(__ldg((k < kWide ? bs : cs).at(row) + n)) : 0.f;
    };
    shared_slots<ROWS, kStepThreads>(slot, a.slots, a.rows, row0, flags);
    // all threads, whatever the row: a row of padding is staged as its slot would be
#pragma unroll
    for (int k = tid; k < ROWS * kChannels; k += kStepThreads)
        if (row0 + k / kChannels < a.rows) stage_token(k / kChannels, row0 + k / kChannels, k % kChannels);
#pragma unroll
    for (int k = tid; k < ROWS * 2 * kWide; k += kStepThreads)
        if (row0 + k / (2 * kWide) < a.rows) stage_shared(k / (2 * kWide), row0 + k / (2 * kWide), k % (2 * kWide));
    load_state(a2, a.A + own, true);
#pragma unroll
    for (int j = 0; j < kStepCols; ++j) a2[j] = decay_rate(a2[j]);
    __syncthreads();
    const unsigned found = a.slots != nullptr ? any_flag(flags) : 0;

    // one token: the state moved on, and its output
    const auto step = [&](float (&s)[kStepCols], int i, int row) {
        const float4 t = token[i][mine];
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < kStepCols; j += 4) {
            const float4 bv = *reinterpret_cast<const float4*>(&shared[i][0][n0 + j]);
            const float4 cv = *reinterpret_cast<const float4*>(&shared[i][1][n0 + j]);
            const float b4[4] = {bv.x, bv.y, bv.z, bv.w}, c4[4] = {cv.x, cv.y, cv.z, cv.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s[j + k] = fmaf(decay(t.x, a2[j + k]), s[j + k], t.y * b4[k]);
                y = fmaf(c4[k], s[j + k], y);
            }
        }
#pragma unroll
        for (int o = LPC / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (part == 0 && mine < cb.n)
            static_cast<T*>(a.out)[static_cast<long long>(row) * a.channels + c] = from_f<T>((y + t.w) * t.z);
    };
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        if (row >= a.rows) break;
        if (slot[i] < 0) {
            if (part == 0 && mine < cb.n) static_cast<T*>(a.out)[static_cast<long long>(row) * a.channels + c] = from_f<T>(0.f);
            continue;
        }
        if (found & (1u << i)) continue;  // the first row with this slot takes them all
        step(h[i], i, row);
        if (found & (0x10000u << i))
            for (int r = row + 1; r < a.rows; ++r)
                if (a.slots[r] == slot[i]) {
                    __syncthreads();  // the same for the whole CTA
                    for (int k = tid; k < kChannels; k += kStepThreads) stage_token(i, r, k);
                    for (int k = tid; k < 2 * kWide; k += kStepThreads) stage_shared(i, r, k);
                    __syncthreads();
                    step(h[i], i, r);
                }
        float* dst = a.state_out + static_cast<long long>(slot[i]) * a.state_out_stride + own;
        if constexpr (VECTOR) {
            if (nn > 0) store8(dst, h[i]);
        } else {
#pragma unroll
            for (int j = 0; j < kStepCols; ++j)
                if (j < nn) dst[j] = h[i][j];
        }
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
    if (!row_steps(a.x_stride, a.dt_stride, a.z_stride, a.b_strides[0], a.c_strides[0]) || a.state_stride < 0 || a.state_out_stride < 0)
        return SSD_ERR_RANGE;
    if (!a.x || !a.dt || !a.A || !a.bm || !a.cm || !a.state || !a.state_out || !a.out) return SSD_ERR_NULL;
    const bool vector = a.dstate % kStepCols == 0 && aligned_to(32, a.A, a.state, a.state_out) &&
                        multiple_of(a.state_stride, kStepCols) && multiple_of(a.state_out_stride, kStepCols);
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const auto with_rows = [&](auto lpc) {
            constexpr int LPC = decltype(lpc)::value;
            const ScanBlocks b = scan_blocks(a.channels, a.groups, kStepThreads / LPC);
            // several rows of a thread share A; one where that would leave SMs without a CTA
            const int rows = static_cast<long long>(a.rows) * b.count(a.groups) >= 16LL * sm_count() ? 4 : 1;
            const dim3 grid((a.rows + rows - 1) / rows, b.count(a.groups));
            if (grid.y > 65535u) return static_cast<int>(SSD_ERR_RANGE);
            const auto launch = [&](auto kernel) {
                launch_plain(kernel, grid, kStepThreads, 0, reinterpret_cast<cudaStream_t>(stream), a, b);
            };
            if (rows > 1)
                vector ? launch(selective_step_kernel<T, LPC, 4, true>) : launch(selective_step_kernel<T, LPC, 4, false>);
            else
                vector ? launch(selective_step_kernel<T, LPC, 1, true>) : launch(selective_step_kernel<T, LPC, 1, false>);
            return launch_status();
        };
        if (a.dstate <= 8) return with_rows(std::integral_constant<int, 1>{});
        if (a.dstate <= 16) return with_rows(std::integral_constant<int, 2>{});
        if (a.dstate <= 32) return with_rows(std::integral_constant<int, 4>{});
        if (a.dstate <= 64) return with_rows(std::integral_constant<int, 8>{});
        return with_rows(std::integral_constant<int, 16>{});
    });
}
