// Short causal convolution along the tokens, one filter of 2 to 4 taps per channel, for batches and packed sequences, its
// gradients, and the step of one token:
//
//   pre[t] = bias + sum_k w[k] in[t - (W-1) + k] ;  out = pre sigmoid(pre) or pre
//   dpre = dout silu'(pre) ;  din[t] = sum_k w[k] dpre[t + (W-1) - k] ;  dw[k] = sum_t dpre[t] in[t - (W-1) + k]
//
// What bounds it: HBM.  A thread owns V neighbouring channels and walks an item of consecutive tokens with the last W
// inputs in registers, the loads of the next kConvAhead tokens in flight; lanes lie along the channels.  An item reads W-1 tokens of
// the one before it again (out of L2).
#include "ssd_vec.cuh"

namespace ssd {

namespace {

constexpr int kConvThreads = 128;
constexpr int kConvVec = 4;  // channels of a thread: 8 or 16 bytes, a row of filters and inputs in registers for each
constexpr int kConvAhead = 4;
// Forward, 16 bits: the tokens ahead are copied into shared memory, kConvRing times kConvAhead of them, which leaves registers for
// six CTAs per SM instead of four: 36.0 us against 38.4 for 8191 packed tokens of 4096 channels.  In fp32 the copies are
// twice as long and cost more than they save: 16.4 against 14.3 us for [4,4096,512].
constexpr int kConvRing = 3;
template <class T, bool VECTOR>
constexpr bool kConvRinged = VECTOR && sizeof(T) == 2;

struct ConvDims {
    SeqMap map;
    int channel_blocks;
};

// The filters of a CTA's channels, through shared memory: in global memory a channel's taps lie side by side, so that a
// thread's own loads would touch a line for each of its channels and taps.
template <class T, int V, int W>
struct Filter {
    static constexpr int kChannels = kConvThreads * V, kRow = kChannels + 8;
    float w[W][V], bias[V];
    __device__ __forceinline__ void load(const void* weight, const void* biases, int f32, int channels, int first) {
        __shared__ __align__(16) float staged[(W + 1) * kRow];
        const int n = min(channels - first, kChannels);
        if (W == 4 && f32 && (reinterpret_cast<uintptr_t>(weight) & 15) == 0) {
            for (int i = threadIdx.x; i < n; i += kConvThreads) {
                const float4 t = __ldg(static_cast<const float4*>(weight) + first + i);
                staged[i] = t.x, staged[kRow + i] = t.y, staged[2 * kRow + i] = t.z, staged[3 * kRow + i] = t.w;
            }
        } else {
            for (int i = threadIdx.x; i < n * W; i += kConvThreads)
                staged[i % W * kRow + i / W] = load_param<T>(weight, f32, static_cast<long long>(first) * W + i);
        }
        for (int i = threadIdx.x; i < n; i += kConvThreads)
            staged[W * kRow + i] = biases != nullptr ? load_param<T>(biases, f32, first + i) : 0.f;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int at = threadIdx.x * V + j;
            const bool in = at < n;
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][j] = in ? staged[k * kRow + at] : 0.f;
            bias[j] = in ? staged[W * kRow + at] : 0.f;
        }
    }
};

// Input of the sequence at t in [-(W-1), len): of the initial state where t < 0.
template <class T, int V, int W, bool VECTOR>
__device__ __forceinline__ void load_input(float (&f)[V], const SsdConvArgs& a, const SeqMap& m, const Span& s, int t, int c,
                                           int n) {
    if (t >= 0) {
        load_f<VECTOR>(f, static_cast<const T*>(a.x) + token_row(m, s, a.batch_stride, a.token_stride, t) + c, n);
    } else if (a.initial_state != nullptr) {
        load_f<VECTOR>(f, static_cast<const T*>(a.initial_state) +
                              (static_cast<long long>(s.seq) * (W - 1) + (t + W - 1)) * a.channels + c, n);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = 0.f;
    }
}

template <class T, int V, int W, bool VECTOR>
__global__ void __launch_bounds__(kConvThreads)
conv_fwd_kernel(const SsdConvArgs a, const ConvDims d) {
    const long long item = blockIdx.x / d.channel_blocks;
    const int c = (blockIdx.x % d.channel_blocks * kConvThreads + threadIdx.x) * V;
    Span s;
    if (!locate(d.map, item, s)) return;
    const int n = max(min(a.channels - c, V), 0);
    T* out = static_cast<T*>(a.out) + ((d.map.cu == nullptr ? s.seq * d.map.tokens : 0) + s.origin) * a.channels + c;
    if (s.pad) {
        const float zero[V] = {};
        for (int t = s.t0; t < s.t1; ++t) store_f<VECTOR>(out + static_cast<long long>(t) * a.channels, zero, n);
        return;
    }
    const Rows<T> x(static_cast<const T*>(a.x) + token_row(d.map, s, a.batch_stride, a.token_stride, 0) + c, a.token_stride);
    const Rows<T> outs(out, a.channels);
    // Each thread copies what it will read itself, so that its own wait is all there is to wait for.
    constexpr bool kRinged = kConvRinged<T, VECTOR>;
    __shared__ Pack<T, V> ring[kRinged ? kConvRing : 1][kConvAhead][kRinged ? kConvThreads : 1];
    Pack<T, V> next[kConvAhead];
    const auto request = [&](int t, int place) {
#pragma unroll
        for (int i = 0; i < kConvAhead; ++i) {
            if constexpr (kRinged)
                copy_async(ring[place][i][threadIdx.x], x.at(min(t + i, s.t1 - 1)), t + i < s.t1 && n > 0);
            else
                load_raw<VECTOR, false>(next[i], x.at(t + i), t + i < s.t1 ? n : 0);
        }
        if (kRinged) copies_commit();
    };
    int place = 0;  // of the tokens at hand
    request(s.t0, 0);
    if (kRinged) {
#pragma unroll
        for (int i = 1; i + 1 < kConvRing; ++i) request(s.t0 + i * kConvAhead, i);
    }
    Filter<T, V, W> f;
    f.load(a.weight, a.bias, a.weight_f32, a.channels, c - threadIdx.x * V);
    float held[W][V];  // the last W inputs, held[W-1] the newest
#pragma unroll
    for (int k = 1; k < W; ++k) load_input<T, V, W, VECTOR>(held[k], a, d.map, s, s.t0 - W + k, c, n);
    for (int t = s.t0; t < s.t1; t += kConvAhead) {
        Pack<T, V> now[kConvAhead];
#pragma unroll
        for (int i = 0; i < kConvAhead; ++i) now[i] = next[i];
        if constexpr (kRinged) {
            copies_wait<kConvRing - 2>();
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) now[i] = ring[place][i][threadIdx.x];
            request(t + (kConvRing - 1) * kConvAhead, place == 0 ? kConvRing - 1 : place - 1);
            place = place + 1 == kConvRing ? 0 : place + 1;
        } else if (t + kConvAhead < s.t1) {
            request(t + kConvAhead, 0);
        }
#pragma unroll
        for (int i = 0; i < kConvAhead; ++i) {
            float o[V], v[V];
            unpack(v, now[i]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
#pragma unroll
                for (int k = 0; k + 1 < W; ++k) held[k][j] = held[k + 1][j];
                held[W - 1][j] = v[j];
                float p = f.bias[j];
#pragma unroll
                for (int k = 0; k < W; ++k) p = fmaf(f.w[k][j], held[k][j], p);
                o[j] = a.silu ? p * sigmoid_fast(p) : p;
            }
            store_f<VECTOR>(outs.to(t + i), o, t + i < s.t1 ? n : 0);
        }
    }
    if (s.last && a.final_state != nullptr) {
        T* fin = static_cast<T*>(a.final_state) + static_cast<long long>(s.seq) * (W - 1) * a.channels + c;
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) {
            float v[V];
            load_input<T, V, W, VECTOR>(v, a, d.map, s, s.len - (W - 1) + k, c, n);
            store_f<VECTOR>(fin + static_cast<long long>(k) * a.channels, v, n);
        }
    }
}

// Items are dealt to the CTAs of a channel block at a distance, so that a thread keeps its channels and sums their share of
// dw in registers; each CTA leaves one row of `work` [CTAs][W + 1][channels], which conv_dw_kernel sums in a fixed order.
// At token t the thread has dpre[t - (W-1) .. t], which is what the gradient of input t - (W-1) takes; the item's last
// W-1 inputs take W-1 tokens of the next one, and the first item's walk starts W-1 inputs early, in the initial state.
template <class T, int V, int W, bool VECTOR>
__global__ void __launch_bounds__(kConvThreads)
conv_bwd_kernel(const SsdConvGradArgs g, const ConvDims d, int slices) {
    const SsdConvArgs& a = g.forward;
    const int slice = blockIdx.x / d.channel_blocks;
    const int c = (blockIdx.x % d.channel_blocks * kConvThreads + threadIdx.x) * V;
    const int n = max(min(a.channels - c, V), 0);
    Filter<T, V, W> f;
    f.load(a.weight, a.bias, a.weight_f32, a.channels, c - threadIdx.x * V);
    float dw[W][V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        db[j] = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][j] = 0.f;
    }
    const long long items = d.map.items();
    for (long long item = slice; item < items; item += slices) {
        Span s;
        if (!locate(d.map, item, s) || n == 0) continue;
        const long long first_row = (d.map.cu == nullptr ? s.seq * d.map.tokens : 0) + s.origin;
        T* dx = static_cast<T*>(g.dx) + first_row * a.channels + c;
        const T* dout = static_cast<const T*>(g.dout) + first_row * a.channels + c;
        if (s.pad) {
            const float zero[V] = {};
            for (int t = s.t0; t < s.t1; ++t) store_f<VECTOR>(dx + static_cast<long long>(t) * a.channels, zero, n);
            continue;
        }
        const Rows<T> x(static_cast<const T*>(a.x) + token_row(d.map, s, a.batch_stride, a.token_stride, 0) + c, a.token_stride);
        const Rows<T> douts(dout, a.channels), dxs(dx, a.channels);
        float held[W][V], dpre[W][V];
#pragma unroll
        for (int k = 1; k < W; ++k) {
            load_input<T, V, W, VECTOR>(held[k], a, d.map, s, s.t0 - W + k, c, n);
#pragma unroll
            for (int j = 0; j < V; ++j) dpre[k][j] = 0.f;
        }
        Pack<T, V> xn[kConvAhead], dn[kConvAhead];
        const int end = min(s.t1 + W - 1, s.len);
        const auto request = [&](int t) {
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) {
                const int in = t + i < end ? n : 0;
                load_raw<VECTOR, false>(xn[i], x.at(t + i), in);
                load_raw<VECTOR, false>(dn[i], douts.at(t + i), in);
            }
        };
        request(s.t0);
        for (int t = s.t0; t < s.t1 + W - 1; t += kConvAhead) {
            Pack<T, V> xr[kConvAhead], dr[kConvAhead];
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) xr[i] = xn[i], dr[i] = dn[i];
            if (t + kConvAhead < s.t1 + W - 1) request(t + kConvAhead);
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) {
                float xs[V], ds[V];
                unpack(xs, xr[i]);
                unpack(ds, dr[i]);
                const int to = t + i - (W - 1);  // the input whose gradient is complete with this token
                const bool mine = t + i < s.t1, there = t + i < end;
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
#pragma unroll
                    for (int k = 0; k + 1 < W; ++k) held[k][j] = held[k + 1][j], dpre[k][j] = dpre[k + 1][j];
                    held[W - 1][j] = xs[j];
                    float e = ds[j];
                    if (a.silu) {
                        float p = f.bias[j];
#pragma unroll
                        for (int k = 0; k < W; ++k) p = fmaf(f.w[k][j], held[k][j], p);
                        const float gate = sigmoid_fast(p);
                        // behind the sequence's end there is no gradient, and what is still held of it may make 0 * inf
                        e = there ? e * gate * fmaf(p, 1.f - gate, 1.f) : 0.f;
                    }
                    dpre[W - 1][j] = e;
                    if (mine) {
                        db[j] += e;
#pragma unroll
                        for (int k = 0; k < W; ++k) dw[k][j] = fmaf(e, held[k][j], dw[k][j]);
                    }
                    float sum = 0.f;
#pragma unroll
                    for (int k = 0; k < W; ++k) sum = fmaf(f.w[k][j], dpre[W - 1 - k][j], sum);
                    o[j] = sum;
                }
                if (to >= s.t1 || (to < s.t0 && !s.first)) continue;
                const int kept = to - (s.len - (W - 1));  // this input is row `kept` of the final state
                if (kept >= 0 && g.dfinal != nullptr) {
                    float df[V];
                    load_f<VECTOR>(df, static_cast<const T*>(g.dfinal) +
                                           (static_cast<long long>(s.seq) * (W - 1) + kept) * a.channels + c, n);
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] += df[j];
                }
                if (to >= 0)
                    store_f<VECTOR>(dxs.to(to), o, n);
                else if (g.dinitial != nullptr)
                    store_f<VECTOR>(static_cast<T*>(g.dinitial) +
                                        (static_cast<long long>(s.seq) * (W - 1) + (to + W - 1)) * a.channels + c, o, n);
            }
        }
    }
    if (g.dweight == nullptr) return;
    float* row = g.work + static_cast<long long>(slice) * (W + 1) * a.channels + c;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (j >= n) break;
#pragma unroll
        for (int k = 0; k < W; ++k) row[static_cast<long long>(k) * a.channels + j] = dw[k][j];
        row[static_cast<long long>(W) * a.channels + j] = db[j];
    }
}

template <class T>
__global__ void __launch_bounds__(kSumCols * kSumRows)
conv_dw_kernel(const float* table, long long rows, int channels, int width, void* dweight, void* dbias, int f32) {
    column_sums(table, rows, static_cast<long long>(channels) * (width + 1), [&](long long col, float v) {
        const long long k = col / channels, c = col - k * channels;
        if (k < width)
            store_param<T>(dweight, f32, c * width + k, v);
        else if (dbias != nullptr)
            store_param<T>(dbias, f32, c, v);
    });
}

// A generation step: the state and the token in, the state moved on by one and the output out.  A thread owns V channels
// of ROWS rows, whose loads are all in flight together, and their filters.  Rows that name the same slot are one another's
// successors: the first of them does the work of all, each taking the inputs that the one before it left, so that nothing
// depends on the order of the CTAs.
template <class T, int V, int W, int ROWS, bool VECTOR>
__global__ void __launch_bounds__(kConvThreads)
conv_step_kernel(const SsdConvStepArgs a, int channel_blocks) {
    __shared__ unsigned flags[kConvThreads / 32];  // see shared_slots
    const int row0 = blockIdx.x / channel_blocks * ROWS;
    const int c = (blockIdx.x % channel_blocks * kConvThreads + threadIdx.x) * V;
    const int n = max(min(a.channels - c, V), 0);
    int slot[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        slot[i] = row >= a.rows ? -1 : a.slots != nullptr ? a.slots[row] : row;
        if (slot[i] >= a.slot_count) slot[i] = -1;
    }
    Pack<T, V> raw[ROWS][W];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int in = slot[i] >= 0 ? n : 0;
        const T* state = static_cast<const T*>(a.state) + (in ? static_cast<long long>(slot[i]) * a.state_stride + c : 0);
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) load_raw<VECTOR, true>(raw[i][k], state + static_cast<long long>(k) * a.channels, in);
        load_raw<VECTOR, false>(raw[i][W - 1], static_cast<const T*>(a.x) + (in ? (row0 + i) * a.x_stride + c : 0), in);
    }
    shared_slots<ROWS, kConvThreads>(slot, a.slots, a.rows, row0, flags);
    Filter<T, V, W> f;
    f.load(a.weight, a.bias, a.weight_f32, a.channels, c - threadIdx.x * V);
    const unsigned found = a.slots != nullptr ? any_flag(flags) : 0;
    auto token = [&](const Pack<T, V> (&held)[W], int row) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float p = f.bias[j];
#pragma unroll
            for (int k = 0; k < W; ++k) p = fmaf(f.w[k][j], to_f(held[k].v[j]), p);
            o[j] = a.silu ? p * sigmoid_fast(p) : p;
        }
        store_f<VECTOR>(static_cast<T*>(a.out) + static_cast<long long>(row) * a.channels + c, o, n);
    };
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        if (row >= a.rows) break;
        if (slot[i] < 0) {
            const float zero[V] = {};
            store_f<VECTOR>(static_cast<T*>(a.out) + static_cast<long long>(row) * a.channels + c, zero, n);
            continue;
        }
        if (found & (1u << i)) continue;  // the first row with this slot takes them all
        token(raw[i], row);
        if (found & (0x10000u << i))
            for (int r = row + 1; r < a.rows; ++r)
                if (a.slots[r] == slot[i]) {
#pragma unroll
                    for (int k = 0; k + 1 < W; ++k) raw[i][k] = raw[i][k + 1];
                    load_raw<VECTOR, false>(raw[i][W - 1], static_cast<const T*>(a.x) + r * a.x_stride + c, n);
                    token(raw[i], r);
                }
        T* next = static_cast<T*>(a.state_out) + static_cast<long long>(slot[i]) * a.state_out_stride + c;
#pragma unroll
        for (int k = 1; k < W; ++k) store_raw<VECTOR>(next + static_cast<long long>(k - 1) * a.channels, raw[i][k], n);
    }
}

int conv_check(const SsdConvArgs& a) {
    if (a.rows <= 0 || a.tokens < 0 || (a.tokens == 0 && a.cu_seqlens == nullptr) || a.channels <= 0 || a.batch_stride < 0 ||
        a.token_stride < 0)
        return SSD_ERR_SHAPE;
    if (a.width < 2 || a.width > 4) return SSD_ERR_UNSUPPORTED;
    if (a.tokens > 0x7fffffff - (1 << 20) || a.rows > 0x7ffffff0 || !row_steps(a.token_stride, a.channels)) return SSD_ERR_RANGE;
    if ((a.tokens > 0 && !a.x) || !a.weight) return SSD_ERR_NULL;
    return SSD_OK;
}
template <class F>
int with_width(int width, F f) {
    switch (width) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        default: return f(std::integral_constant<int, 4>{});
    }
}
// Tokens of an item, so that the items are the CTAs that the SMs hold at a time, `resident` each: the filters are staged and
// the W-1 tokens in front read once for as many tokens as that allows.
int conv_span(const SsdConvArgs& a, int channel_blocks, int resident, int least) {
    const long long ctas = (static_cast<long long>(resident) * sm_count() + channel_blocks - 1) / channel_blocks;
    const long long sequences = a.cu_seqlens ? 1 : a.rows, per = ctas > sequences ? ctas / sequences : 1;
    const long long span = (a.tokens + per - 1) / per;
    return static_cast<int>(span < least ? least : span);
}
// Backward, those CTAs (three per SM, by registers) are dealt one item each where the sequences allow.
constexpr int kConvCtas = 4, kConvRingedCtas = 6, kConvGradCtas = 3;
ConvDims conv_grad_dims(const SsdConvArgs& a) {
    const int blocks = (a.channels + kConvThreads * kConvVec - 1) / (kConvThreads * kConvVec);
    return ConvDims{{a.cu_seqlens, a.tokens, a.rows, conv_span(a, blocks, kConvGradCtas, 16)}, blocks};
}
int conv_slices(const ConvDims& d) {
    const long long items = d.map.items(), fill = (static_cast<long long>(kConvGradCtas) * sm_count() + d.channel_blocks - 1) / d.channel_blocks;
    return static_cast<int>(items < fill ? items : fill);
}

}  // namespace

}  // namespace ssd

extern "C" int ssd_short_conv_fwd(const SsdConvArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdConvArgs& a = *args;
    if (const int rc = conv_check(a); rc != SSD_OK) return rc;
    if (!a.out && a.tokens > 0) return SSD_ERR_NULL;
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = kConvVec;
        const int channel_blocks = (a.channels + kConvThreads * V - 1) / (kConvThreads * V);
        const bool vector = aligned_to(sizeof(T) * V, a.x, a.initial_state, a.out, a.final_state) && multiple_of(a.channels, V) &&
                            multiple_of(a.batch_stride, V) && multiple_of(a.token_stride, V);
        const int ctas = vector && kConvRinged<T, true> ? kConvRingedCtas : kConvCtas;
        const ConvDims d{{a.cu_seqlens, a.tokens, a.rows, conv_span(a, channel_blocks, ctas, 8)}, channel_blocks};
        const long long blocks = d.map.items() * channel_blocks;
        if (blocks > 0x7fffffffLL) return static_cast<int>(SSD_ERR_RANGE);
        return with_width(a.width, [&](auto w) {
            constexpr int W = decltype(w)::value;
            launch_plain(vector ? conv_fwd_kernel<T, V, W, true> : conv_fwd_kernel<T, V, W, false>, static_cast<unsigned>(blocks),
                         kConvThreads, 0, reinterpret_cast<cudaStream_t>(stream), a, d);
            return launch_status();
        });
    });
}

extern "C" size_t ssd_short_conv_work_bytes(const SsdConvArgs* args) {
    using namespace ssd;
    if (args == nullptr || conv_check(*args) != SSD_OK) return 0;
    return sizeof(float) * conv_slices(conv_grad_dims(*args)) * static_cast<size_t>(args->width + 1) * args->channels;
}

extern "C" int ssd_short_conv_bwd(const SsdConvGradArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdConvGradArgs& g = *args;
    const SsdConvArgs& a = g.forward;
    if (const int rc = conv_check(a); rc != SSD_OK) return rc;
    if ((a.tokens > 0 && (!g.dout || !g.dx)) || (g.dweight && !g.work) || (g.dbias && !g.dweight)) return SSD_ERR_NULL;
    const ConvDims d = conv_grad_dims(a);
    const int slices = conv_slices(d);
    const long long blocks = static_cast<long long>(slices) * d.channel_blocks;
    if (blocks > 0x7fffffffLL) return SSD_ERR_RANGE;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = kConvVec;
        const bool vector = aligned_to(sizeof(T) * V, a.x, a.initial_state, g.dout, g.dfinal, g.dx, g.dinitial) &&
                            multiple_of(a.channels, V) && multiple_of(a.batch_stride, V) && multiple_of(a.token_stride, V);
        const int rc = with_width(a.width, [&](auto w) {
            constexpr int W = decltype(w)::value;
            launch_plain(vector ? conv_bwd_kernel<T, V, W, true> : conv_bwd_kernel<T, V, W, false>, static_cast<unsigned>(blocks),
                         kConvThreads, 0, st, g, d, slices);
            return launch_status();
        });
        if (rc != SSD_OK || g.dweight == nullptr) return rc;
        const long long cols = static_cast<long long>(a.channels) * (a.width + 1);
        launch_plain(conv_dw_kernel<T>, static_cast<unsigned>((cols + kSumCols - 1) / kSumCols), kSumCols * kSumRows, 0, st, g.work,
                     static_cast<long long>(slices), a.channels, a.width, g.dweight, g.dbias, a.weight_f32);
        return launch_status();
    });
}

extern "C" int ssd_short_conv_step(const SsdConvStepArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdConvStepArgs& a = *args;
    if (a.rows <= 0 || a.channels <= 0 || a.slot_count <= 0 || a.x_stride < 0 || a.state_stride < 0 || a.state_out_stride < 0 ||
        (a.slots == nullptr && a.slot_count < a.rows))
        return SSD_ERR_SHAPE;
    if (a.width < 2 || a.width > 4) return SSD_ERR_UNSUPPORTED;
    if (!a.x || !a.weight || !a.state || !a.state_out || !a.out) return SSD_ERR_NULL;
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = kConvVec;
        const int channel_blocks = (a.channels + kConvThreads * V - 1) / (kConvThreads * V);
        // several rows share the filters; one where that would leave SMs without a CTA
        const int rows = static_cast<long long>(a.rows) * channel_blocks >= 8LL * sm_count() ? 4 : 1;
        const long long blocks = static_cast<long long>((a.rows + rows - 1) / rows) * channel_blocks;
        if (blocks > 0x7fffffffLL) return static_cast<int>(SSD_ERR_RANGE);
        const bool vector = aligned_to(sizeof(T) * V, a.x, a.state, a.state_out, a.out) && multiple_of(a.channels, V) &&
                            multiple_of(a.x_stride, V) && multiple_of(a.state_stride, V) && multiple_of(a.state_out_stride, V);
        return with_width(a.width, [&](auto w) {
            constexpr int W = decltype(w)::value;
            const auto launch = [&](auto kernel) {
                launch_plain(kernel, static_cast<unsigned>(blocks), kConvThreads, 0, reinterpret_cast<cudaStream_t>(stream), a,
                             channel_blocks);
            };
            if (rows > 1)
                vector ? launch(conv_step_kernel<T, V, W, 4, true>) : launch(conv_step_kernel<T, V, W, 4, false>);
            else
                vector ? launch(conv_step_kernel<T, V, W, 1, true>) : launch(conv_step_kernel<T, V, W, 1, false>);
            return launch_status();
        });
    });
}
