// Root-mean-square norm with the residual's addition, its gradients, and the same norm with an output in 8 bits:
//
//   v = x + residual ;  r = (mean(v^2) + eps)^-1/2 ;  out = v r w              q = e4m3(out / s), s = max|out| / 448 per row or group
//   g = dout w ;  dv = r (g - v r mean(g v r)) + dstream ;  dw = sum_rows dout v r
//
// What bounds them: HBM.  Each element is loaded once, held in registers as fp32 between the row's sum and the output, and
// stored once.  A thread owns vectors of 16 bytes (`VEC` elements), ITER of them, `tpr` threads make a row: rows of up to 4
// vectors per lane are a warp's, longer ones a CTA's.  Scalar loads take the same elements where rows are not aligned.
#include <cuda_fp8.h>

#include "ssd_vec.cuh"

namespace ssd {

namespace {

constexpr int kNormMaxWidth = 16384;
constexpr int kNormThreads = 512;
constexpr long long kNormMaxRows = 0x7fffffff - (1 << 20);  // a walk's step behind the last is still a number

template <class T>
constexpr int kNormVec = 16 / static_cast<int>(sizeof(T));

// Sums and maxima over the tpr threads of a row; `part` has room for 2 x 16 floats per call site.
struct Reduced {
    float sum, top;
};
template <bool TOP>
__device__ __forceinline__ Reduced reduce_row(float sum, float top, int tpr, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (TOP) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (tpr > 32) {  // then the row is the whole CTA's
        const int warp = threadIdx.x >> 5, warps = tpr >> 5, lane = threadIdx.x & 31;
        if (lane == 0) {
            part[warp] = sum;
            if (TOP) part[16 + warp] = top;
        }
        __syncthreads();
        // at most 16 warps
        sum = (lane & 15) < warps ? part[lane & 15] : 0.f;
        if (TOP) top = (lane & 15) < warps ? part[16 + (lane & 15)] : 0.f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (TOP) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
    }
    return {sum, top};
}

enum NormOut { kPlain, kRowScale, kGroupScale, kOneScale };

template <class T, class R, int ITER, bool VECTOR, NormOut kOut>
__global__ void __launch_bounds__(kNormThreads)
norm_fwd_kernel(const SsdNormArgs a, int tpr) {
    constexpr int VEC = kNormVec<T>;
    __shared__ float part[32];
    const int at = tpr == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int row = tpr == 32 ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const bool live = row < a.rows;
    const T* x = Rows<T>(static_cast<const T*>(a.x), a.x_stride).at(row);
    const R* res = Rows<R>(static_cast<const R*>(a.residual), a.residual_stride).at(row);
    Pack<T, VEC> xr[ITER];
    Pack<R, VEC> rr[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (at + i * tpr) * VEC, n = live ? min(a.width - c, VEC) : 0;
        load_raw<VECTOR, false>(xr[i], x + c, n);
        if (a.residual != nullptr) load_raw<VECTOR, false>(rr[i], res + c, n);
    }
    float v[ITER][VEC], w[ITER][VEC];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (at + i * tpr) * VEC, n = min(a.width - c, VEC);
        if (a.weight_f32)
            load_f<VECTOR>(w[i], static_cast<const float*>(a.weight) + c, n);
        else
            load_f<VECTOR>(w[i], static_cast<const T*>(a.weight) + c, n);
    }
    float sum = 0.f, top = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (at + i * tpr) * VEC, n = live ? min(a.width - c, VEC) : 0;
        unpack(v[i], xr[i]);
        if (a.residual != nullptr) {
            float r[VEC];
            unpack(r, rr[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] += r[j];
            store_f<VECTOR>(Rows<R>(static_cast<R*>(a.stream), a.width).to(row) + c, v[i], n);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            sum = fmaf(v[i][j], v[i][j], sum);
            if (kOut == kRowScale) top = max_nan(top, fabsf(v[i][j] * w[i][j]));
        }
    }
    const Reduced red = reduce_row<kOut == kRowScale>(sum, top, tpr, part);
    const float rstd = rsqrtf(red.sum / static_cast<float>(a.width) + a.eps);
    if (a.rstd != nullptr && live && at == 0) a.rstd[row] = rstd;
    if constexpr (kOut == kPlain) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (at + i * tpr) * VEC, n = live ? min(a.width - c, VEC) : 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] = v[i][j] * rstd * w[i][j];
            store_f<VECTOR>(Rows<T>(static_cast<T*>(a.out), a.width).to(row) + c, v[i], n);
        }
    } else {
        float scale = 1.f;
        if (kOut == kOneScale) scale = *static_cast<const float*>(a.static_scale);
        if (kOut == kRowScale) {
            // rstd is positive, so the largest |v w| is the largest |out| but for rstd
            scale = red.top * rstd * (1.f / 448.f);
            if (scale == 0.f) scale = 1.f;
            if (live && at == 0) a.scales[row] = scale;
        }
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (at + i * tpr) * VEC, n = live ? min(a.width - c, VEC) : 0;
            float y[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) y[j] = v[i][j] * rstd * w[i][j];
            if (kOut == kGroupScale) {
                // a group is group / VEC neighbouring lanes, a power of two that divides 32
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < VEC; ++j) m = max_nan(m, fabsf(y[j]));
                for (int o = a.group / VEC / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                scale = m * (1.f / 448.f);
                if (scale == 0.f) scale = 1.f;
                const int lg = 31 - __clz(a.group);
                if (n > 0 && (c & (a.group - 1)) == 0) a.scales[static_cast<long long>(row) * (a.width >> lg) + (c >> lg)] = scale;
            }
            // times the reciprocal (one step off at most), but for scales so small that it would overflow
            if (fabsf(scale) < 1e-30f) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[j] = y[j] / scale;
            } else {
                const float inv = rcpf(scale);
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[j] *= inv;
            }
            alignas(8) unsigned char q[VEC];
#pragma unroll
            for (int j = 0; j < VEC; j += 4)
                *reinterpret_cast<unsigned*>(q + j) =
                    __nv_cvt_float2_to_fp8x2(make_float2(y[j], y[j + 1]), __NV_SATFINITE, __NV_E4M3) |
                    static_cast<unsigned>(__nv_cvt_float2_to_fp8x2(make_float2(y[j + 2], y[j + 3]), __NV_SATFINITE, __NV_E4M3)) << 16;
            unsigned char* dst = Rows<unsigned char>(static_cast<unsigned char*>(a.q), a.width).to(row) + c;
            if constexpr (VECTOR) {
                using B = typename Bits<VEC>::type;
                if (n > 0) *reinterpret_cast<B*>(dst) = *reinterpret_cast<B*>(q);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (j < n) dst[j] = q[j];
            }
        }
    }
}

// CTAs walk the rows at a distance of the grid, so that a thread keeps its columns and sums their share of dw in registers;
// the CTA's rows are added up in shared memory and leave as one row of `work`, which norm_dw_kernel sums in a fixed order.
// The next row's loads are in flight under this one's sums.
template <class T, class R, int ITER, bool VECTOR>
__global__ void __launch_bounds__(kNormThreads, ITER == 1 ? 2 : 1)
norm_bwd_kernel(const SsdNormGradArgs a, int tpr) {
    constexpr int VEC = kNormVec<T>;
    __shared__ float part[2][32];
    extern __shared__ float norm_rows[];  // [rows of the CTA][width], only where there are several
    const int at = tpr == 32 ? threadIdx.x & 31 : threadIdx.x, mine = tpr == 32 ? threadIdx.x >> 5 : 0;
    const int rows_here = tpr == 32 ? blockDim.x >> 5 : 1;
    float dw[ITER][VEC];
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) dw[i][j] = 0.f;
    Pack<R, VEC> vr[ITER], sr[ITER];
    Pack<T, VEC> gr[ITER], ur[ITER];
    float rstd_next = 0.f;
    const Rows<R> streams(static_cast<const R*>(a.stream), a.stream_stride), dstreams(static_cast<const R*>(a.dstream), a.dstream_stride);
    const Rows<T> douts(static_cast<const T*>(a.dout), a.dout_stride), addends(static_cast<const T*>(a.addend), a.addend_stride);
    const Rows<T> dxs(static_cast<T*>(a.dx), a.width);
    const Rows<R> dresiduals(static_cast<R*>(a.dresidual), a.width);
    const auto request = [&](int row) {
        const bool live = row < a.rows;
        rstd_next = live ? __ldg(a.rstd + row) : 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (at + i * tpr) * VEC, n = live ? min(a.width - c, VEC) : 0;
            load_raw<VECTOR, false>(vr[i], streams.at(row) + c, n);
            load_raw<VECTOR, false>(gr[i], douts.at(row) + c, n);
            if (a.dstream != nullptr)
                load_raw<VECTOR, false>(sr[i], dstreams.at(row) + c, n);
            if (a.addend != nullptr)
                load_raw<VECTOR, false>(ur[i], addends.at(row) + c, n);
        }
    };
    const int step = gridDim.x * rows_here, count = static_cast<int>(a.rows);
    request(blockIdx.x * rows_here + mine);
    int parity = 0;
    for (int first = blockIdx.x * rows_here; first < count; first += step) {
        const int row = first + mine;
        const bool live = row < a.rows;
        const float rstd = rstd_next;
        float v[ITER][VEC], g[ITER][VEC];
        Pack<R, VEC> s[ITER];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (at + i * tpr) * VEC, n = min(a.width - c, VEC);
            float w[VEC];
            if (a.weight_f32)
                load_f<VECTOR>(w, static_cast<const float*>(a.weight) + c, n);
            else
                load_f<VECTOR>(w, static_cast<const T*>(a.weight) + c, n);
            unpack(v[i], vr[i]);
            unpack(g[i], gr[i]);
            s[i] = sr[i];
            if (a.addend != nullptr) {
                float u[VEC];
                unpack(u, ur[i]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[i][j] += u[j];
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] *= rstd;
                dw[i][j] = fmaf(g[i][j], v[i][j], dw[i][j]);
                g[i][j] *= w[j];
                dot = fmaf(g[i][j], v[i][j], dot);
            }
        }
        if (first + step < count) request(row + step);
        const float mean = reduce_row<false>(dot, 0.f, tpr, part[parity]).sum / static_cast<float>(a.width);
        parity ^= 1;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (at + i * tpr) * VEC, n = live ? min(a.width - c, VEC) : 0;
            float d[VEC] = {};
            if (a.dstream != nullptr) unpack(d, s[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[i][j] = fmaf(rstd, fmaf(-v[i][j], mean, g[i][j]), d[j]);
            store_f<VECTOR>(dxs.to(row) + c, g[i], n);
            if (a.dresidual != nullptr) store_f<VECTOR>(dresiduals.to(row) + c, g[i], n);
        }
    }
    if (a.dweight == nullptr) return;
    float* table = a.work + static_cast<long long>(blockIdx.x) * a.width;
    if (rows_here > 1) {
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int c = (at + i * tpr) * VEC + j;
                if (c < a.width) norm_rows[mine * a.width + c] = dw[i][j];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
            float sum = 0.f;
            for (int k = 0; k < rows_here; ++k) sum += norm_rows[k * a.width + c];
            table[c] = sum;
        }
    } else {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (at + i * tpr) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < a.width) table[c + j] = dw[i][j];
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kSumCols * kSumRows)
norm_dw_kernel(const float* table, long long rows, int width, void* dweight, int f32) {
    column_sums(table, rows, width, [&](long long c, float v) { store_param<T>(dweight, f32, c, v); });
}

struct NormGeometry {
    int tpr, iter, rows_here;
};
// Threads per row and vectors per thread.  Rows of up to 32 vectors per thread's share are a warp's; of longer ones a thread
// takes one vector where there are few rows (latency counts) and up to `most` where they fill the GPU anyway (fewer threads
// to reduce over).
NormGeometry norm_geometry(long long rows, int width, int vec, int most) {
    const int vecs = (width + vec - 1) / vec;
    const bool many = rows >= 8LL * sm_count();
    NormGeometry g{32, 1, 1};
    if (vecs <= 32 * most && (many || vecs <= 32)) {
        g.iter = vecs <= 32 ? 1 : vecs <= 64 ? 2 : 4;
    } else {
        int iter = many ? most : 1;
        while ((vecs + iter - 1) / iter > kNormThreads) iter *= 2;
        g.iter = iter;
        g.tpr = ((vecs + iter - 1) / iter + 31) / 32 * 32;
    }
    g.rows_here = g.tpr == 32 && many ? 8 : 1;
    return g;
}
// Backward: two vectors per thread only where a row is one warp's or would take more than a CTA's threads.
NormGeometry norm_grad_geometry(long long rows, int width, int vec) {
    return norm_geometry(rows, width, vec, (width + vec - 1) / vec <= 64 ? 2 : 1);
}
unsigned norm_bwd_grid(long long rows, const NormGeometry& g) {
    const long long all = (rows + g.rows_here - 1) / g.rows_here;
    const int threads = g.tpr * g.rows_here;
    const long long resident = static_cast<long long>(sm_count()) * ((g.iter == 1 ? 1024 : 512) / threads);
    return static_cast<unsigned>(all < resident ? all : resident);
}

template <class T, class F>
int with_residual_type(int residual_f32, F f) {
    if constexpr (sizeof(T) == 4) {
        return f(T{});
    } else {
        return residual_f32 ? f(float{}) : f(T{});
    }
}
template <class T, class F>
int with_iter(int iter, F f) {
    switch (iter) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        default: return f(std::integral_constant<int, kNormMaxWidth / kNormThreads / kNormVec<T>>{});
    }
}

}  // namespace

}  // namespace ssd

extern "C" int ssd_rms_norm_fwd(const SsdNormArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdNormArgs& a = *args;
    if (a.rows <= 0 || a.width <= 0 || a.x_stride < 0 || a.residual_stride < 0) return SSD_ERR_SHAPE;
    if (a.width > kNormMaxWidth) return SSD_ERR_UNSUPPORTED;
    if (a.rows > kNormMaxRows || !row_steps(a.x_stride, a.residual_stride)) return SSD_ERR_RANGE;
    const bool quant = a.q != nullptr;
    if (!a.x || !a.weight || (!quant && !a.out) || (a.residual && !a.stream) || (quant && !a.static_scale && !a.scales))
        return SSD_ERR_NULL;
    if (a.group != 0 && ((a.group != 32 && a.group != 64 && a.group != 128) || a.width % a.group != 0)) return SSD_ERR_SHAPE;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return with_residual_type<T>(a.residual_f32, [&](auto r) {
            using R = decltype(r);
            const int vec = kNormVec<T>;
            const NormGeometry g = norm_geometry(a.rows, a.width, vec, quant ? 2 : 4);
            const long long blocks = (a.rows + g.rows_here - 1) / g.rows_here;
            if (blocks > 0x7fffffffLL) return static_cast<int>(SSD_ERR_RANGE);
            const bool vector = aligned16(a.x, a.residual, a.weight, a.out, a.stream, a.q) && multiple_of(a.width, vec) &&
                                multiple_of(a.x_stride, vec) && multiple_of(a.residual_stride, vec);
            return with_iter<T>(g.iter, [&](auto it) {
                constexpr int I = decltype(it)::value;
                const auto launch = [&](auto kernel) {
                    launch_plain(kernel, static_cast<unsigned>(blocks), g.tpr * g.rows_here, 0, st, a, g.tpr);
                };
                const auto with = [&](auto out) {
                    constexpr NormOut kOut = decltype(out)::value;
                    vector ? launch(norm_fwd_kernel<T, R, I, true, kOut>) : launch(norm_fwd_kernel<T, R, I, false, kOut>);
                };
                if (!quant)
                    with(std::integral_constant<NormOut, kPlain>{});
                else if (a.static_scale != nullptr)
                    with(std::integral_constant<NormOut, kOneScale>{});
                else if (a.group != 0)
                    with(std::integral_constant<NormOut, kGroupScale>{});
                else
                    with(std::integral_constant<NormOut, kRowScale>{});
                return launch_status();
            });
        });
    });
}

extern "C" size_t ssd_rms_norm_work_bytes(int64_t rows, int width, int dtype) {
    using namespace ssd;
    if (rows <= 0 || width <= 0 || width > kNormMaxWidth || dtype < SSD_F32 || dtype > SSD_F16) return 0;
    const NormGeometry g = norm_grad_geometry(rows, width, dtype == SSD_F32 ? 4 : 8);
    return sizeof(float) * static_cast<size_t>(norm_bwd_grid(rows, g)) * width;
}

extern "C" int ssd_rms_norm_bwd(const SsdNormGradArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdNormGradArgs& a = *args;
    if (a.rows <= 0 || a.width <= 0 || a.dout_stride < 0 || a.dstream_stride < 0 || a.stream_stride < 0 ||
        a.addend_stride < 0) return SSD_ERR_SHAPE;
    if (a.width > kNormMaxWidth) return SSD_ERR_UNSUPPORTED;
    if (a.rows > kNormMaxRows || !row_steps(a.dout_stride, a.dstream_stride, a.stream_stride, a.addend_stride)) return SSD_ERR_RANGE;
    if (!a.dout || !a.stream || !a.weight || !a.rstd || !a.dx || (a.dweight && !a.work)) return SSD_ERR_NULL;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return with_residual_type<T>(a.residual_f32, [&](auto r) {
            using R = decltype(r);
            const int vec = kNormVec<T>;
            const NormGeometry g = norm_grad_geometry(a.rows, a.width, vec);
            const unsigned grid = norm_bwd_grid(a.rows, g);
            const size_t smem = g.rows_here > 1 ? sizeof(float) * g.rows_here * a.width : 0;
            const bool vector = aligned16(a.dout, a.dstream, a.stream, a.addend, a.weight, a.dx, a.dresidual) &&
                                multiple_of(a.width, vec) && multiple_of(a.dout_stride, vec) &&
                                multiple_of(a.dstream_stride, vec) && multiple_of(a.stream_stride, vec) &&
                                multiple_of(a.addend_stride, vec);
            const int rc = with_iter<T>(g.iter, [&](auto it) {
                constexpr int I = decltype(it)::value;
                const auto launch = [&](auto kernel) { launch_plain(kernel, grid, g.tpr * g.rows_here, smem, st, a, g.tpr); };
                vector ? launch(norm_bwd_kernel<T, R, I, true>) : launch(norm_bwd_kernel<T, R, I, false>);
                return launch_status();
            });
            if (rc != SSD_OK || a.dweight == nullptr) return rc;
            launch_plain(norm_dw_kernel<T>, static_cast<unsigned>((a.width + kSumCols - 1) / kSumCols), kSumCols * kSumRows, 0, st,
                         a.work, static_cast<long long>(grid), a.width, a.dweight, a.weight_f32);
            return launch_status();
        });
    });
}
