// Selective scan, gradients.  With dy = dout silu(z) and g the gradient of the states,
//
//   g_t = C_t dy_t + a_{t+1} g_{t+1} ;  dC_t[n] = sum_c dy_t h_t[n] ;  dB_t[n] = sum_c g_t[n] dt_t x_t ;  du_t = sum_n g_t[n] B_t[n]
//   q_t[n] = g_t[n] a_t[n] h_{t-1}[n] ;  ddt_t = x_t du_t + sum_n q_t[n] A[n] ;  dA[n] = sum_t q_t[n] dt_t ;  dx_t = dt_t du_t + D dy_t
//
// What bounds it: about 15 instructions for each (token, channel, state column), a fifth of them the sums of dB and dC over
// the channels, which lie along the lanes.  The bytes are few beside that.
//
// Layout: a lane owns two neighbouring channels (packed arithmetic), a warp kTokens tokens of 64 channels, a CTA a chunk
// of kWarps * kTokens tokens, which it walks from the sequence's end.  For one state column at a time each warp forms its
// exponentials once, runs the recurrences of h and g from zero over its tokens, and puts their ends and the product of its
// decays into shared memory; after one barrier it folds those of the warps before (behind) it into its true start, and
// runs both recurrences again on the exponentials it still holds.  h enters a chunk from the forward pass's checkpoints, g
// from the chunk behind.  Sums over n stay with the thread.  dB and dC replace B and C in shared memory (a warp's tokens are
// its own) and leave as one table per block of channels, summed in a fixed order by scan_shared_sum_kernel.
#include "ssd_selective.cuh"

namespace ssd {

namespace {

constexpr int kWarps = 8, kTokens = 8, kChunk = kWarps * kTokens, kBwdChannels = 64;
static_assert(kChunk == kScanCheckpoint, "a chunk starts from a checkpoint");
constexpr int kRow = kChunk + 4;  // tokens of a state column in shared memory, padded

struct BwdLaunch {
    SeqMap map;
    ScanBlocks blocks;
    bool split;
    const float* ends;    // [items][dstate][channels] gradient of the state behind each segment, where split
    float* shared_part;   // [2][blocks of a group][tokens][groups][dstate]: dB, dC
    float* channel_part;  // [items][dstate + 2][channels]: dA, dD, d_dt_bias
    long long all_tokens;
};

size_t bwd_smem(int dstate) {
    return sizeof(float) * (2 * dstate * kRow + 4 * dstate * kBwdChannels + 2 * kWarps * kBwdChannels * (2 + 1 + 1));
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Sums over the 32 lanes of 16 values each: a lane ends up with the sum of value `lane / 2` (both of a pair the same).  Each
// step hands half of the values to the lane on the other side, 8 + 4 + 2 + 1 + 1 exchanges instead of 80.
__device__ __forceinline__ float sum_lanes16(float (&v)[16], int lane) {
#pragma unroll
    for (int half = 8, bit = 16; half > 0; half >>= 1, bit >>= 1) {
        const bool upper = (lane & bit) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float keep = upper ? v[i + half] : v[i], send = upper ? v[i] : v[i + half];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

template <class T, bool VECTOR, bool GATED>
__global__ void __launch_bounds__(32 * kWarps)
selective_bwd_kernel(const SsdScanGradArgs g, const BwdLaunch l) {
    const SsdScanArgs& a = g.forward;
    extern __shared__ __align__(16) float bwd_smem_[];
    const int N = a.dstate, blocks = l.blocks.count(a.groups);
    const long long item = blockIdx.x / blocks;
    const ChannelBlock cb = channel_block(l.blocks, blockIdx.x % blocks, a.channels, a.groups);
    const int in_group = blockIdx.x % blocks % l.blocks.per_group;
    Span s;
    if (!locate(l.map, item, s)) {
        // nothing of this item, but its row of the table is summed
        for (int i = threadIdx.x; i < (N + 2) * cb.n; i += 32 * kWarps)
            l.channel_part[(item * (N + 2) + i / cb.n) * a.channels + cb.first + i % cb.n] = 0.f;
        return;
    }
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const long long first_token = (l.map.cu == nullptr ? s.seq * l.map.tokens : 0) + s.origin;
    const long long shared_table = l.all_tokens * a.groups * N;
    // dB and dC of this block of channels, by token of all sequences
    float* db = l.shared_part + in_group * shared_table + (first_token * a.groups + cb.group) * N;
    float* dc = db + l.blocks.per_group * shared_table;
    if (s.pad) {
        for (long long i = tid; i < static_cast<long long>(s.t1 - s.t0) * cb.n; i += 32 * kWarps) {
            const long long at = (first_token + s.t0 + i / cb.n) * a.channels + cb.first + i % cb.n;
            static_cast<T*>(g.dx)[at] = from_f<T>(0.f);
            static_cast<T*>(g.ddt)[at] = from_f<T>(0.f);
            if (GATED) static_cast<T*>(g.dz)[at] = from_f<T>(0.f);
        }
        for (long long i = tid; i < static_cast<long long>(s.t1 - s.t0) * N; i += 32 * kWarps) {
            const long long at = (s.t0 + i / N) * a.groups * N + i % N;
            db[at] = dc[at] = 0.f;
        }
        for (int i = tid; i < (N + 2) * cb.n; i += 32 * kWarps)
            l.channel_part[(item * (N + 2) + i / cb.n) * a.channels + cb.first + i % cb.n] = 0.f;
        return;
    }

    float* sb = bwd_smem_;                          // [N][kRow] B, later dB
    float* sc = sb + N * kRow;                      // [N][kRow] C, later dC
    float* sa = sc + N * kRow;                      // [N][64] A log2(e)
    float* sg = sa + N * kBwdChannels;              // [2][N][64] gradient of the state behind the chunk
    float* sda = sg + 2 * N * kBwdChannels;         // [N][64] dA
    float4* ex_h = reinterpret_cast<float4*>(sda + N * kBwdChannels);                   // [2][warps][32] decay, end of h
    float2* ex_g = reinterpret_cast<float2*>(ex_h + 2 * kWarps * 32);                   // [2][warps][32] end of g
    float2* ex_a = ex_g + 2 * kWarps * 32;                                              // [2][warps][32] dA of the warp

    const int c = cb.first + 2 * lane, pn = max(min(cb.n - 2 * lane, 2), 0);
    for (int i = tid; i < N * kBwdChannels; i += 32 * kWarps) {
        const int n = i / kBwdChannels, ch = i % kBwdChannels;
        const bool in = ch < cb.n;
        sa[i] = in ? a.A[static_cast<long long>(cb.first + ch) * N + n] * kLog2e : 0.f;
        sda[i] = 0.f;
        float end = 0.f;
        if (in) {
            if (l.split)
                end = l.ends[(item * N + n) * a.channels + cb.first + ch];
            else if (g.dfinal != nullptr)
                end = g.dfinal[(static_cast<long long>(s.seq) * a.channels + cb.first + ch) * N + n];
        }
        sg[i] = end;
    }
    float2 bias = make_float2(0.f, 0.f), skip = bias, dskip = bias, dbias = bias;
    if (a.dt_bias != nullptr) bias = make_float2(pn > 0 ? a.dt_bias[c] : 0.f, pn > 1 ? a.dt_bias[c + 1] : 0.f);
    if (a.D != nullptr) skip = make_float2(pn > 0 ? a.D[c] : 0.f, pn > 1 ? a.D[c + 1] : 0.f);

    const T* x = static_cast<const T*>(a.x) + token_row(l.map, s, a.x_strides[0], a.x_strides[1], 0) + c;
    const T* dtp = static_cast<const T*>(a.dt) + token_row(l.map, s, a.dt_strides[0], a.dt_strides[1], 0) + c;
    const T* z = static_cast<const T*>(a.z) + token_row(l.map, s, a.z_strides[0], a.z_strides[1], 0) + c;
    const T* bm = static_cast<const T*>(a.bm) + token_row(l.map, s, a.b_strides[0], a.b_strides[1], 0) + cb.group * a.b_strides[2];
    const T* cm = static_cast<const T*>(a.cm) + token_row(l.map, s, a.c_strides[0], a.c_strides[1], 0) + cb.group * a.c_strides[2];
    const T* dout = static_cast<const T*>(g.dout) + first_token * a.channels + c;
    const long long checkpoint0 = l.map.cu == nullptr
                                      ? s.seq * ((l.map.tokens + kScanCheckpoint - 1) / kScanCheckpoint)
                                      : s.origin / kScanCheckpoint + s.seq;

    const int chunks = (s.t1 - s.t0 + kChunk - 1) / kChunk;
    int side = 0;  // of sg
    for (int k = chunks - 1; k >= 0; --k) {
        const int t0 = s.t0 + k * kChunk, tw = t0 + w * kTokens;
        // ---- this warp's tokens
        F2 dt[kTokens], u[kTokens], dy[kTokens];
        float2 sum_dt = make_float2(0.f, 0.f);
        Pack<T, 2> xr[kTokens], dr[kTokens], zr[kTokens], gr[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int t = tw + i, n = t < s.t1 ? pn : 0;
            load_raw<VECTOR, false>(xr[i], x + t * a.x_strides[1], n);
            load_raw<VECTOR, false>(dr[i], dtp + t * a.dt_strides[1], n);
            load_raw<VECTOR, false>(gr[i], dout + static_cast<long long>(t) * a.channels, n);
            if (GATED) load_raw<VECTOR, false>(zr[i], z + t * a.z_strides[1], n);
        }
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const float2 xv = pair_f(xr[i]);
            float2 d = pair_f(dr[i]), o = pair_f(gr[i]);
            d = make_float2(d.x + bias.x, d.y + bias.y);
            if (a.softplus) d = make_float2(softplus_series(d.x), softplus_series(d.y));
            if (tw + i >= s.t1) d = make_float2(0.f, 0.f);
            if (GATED) {
                const float2 zv = pair_f(zr[i]);
                o = make_float2(o.x * zv.x * sigmoid_fast(zv.x), o.y * zv.y * sigmoid_fast(zv.y));
            }
            sum_dt = make_float2(sum_dt.x + d.x, sum_dt.y + d.y);
            dt[i] = pack2(d.x, d.y);
            u[i] = pack2(d.x * xv.x, d.y * xv.y);
            dy[i] = pack2(o.x, o.y);
        }
        for (int i = tid; i < N * kChunk; i += 32 * kWarps) {
            const int t = i / N, n = i % N;
            const bool in = t0 + t < s.t1;
            sb[n * kRow + t] = in ? to_f(bm[(t0 + t) * a.b_strides[1] + n]) : 0.f;
            sc[n * kRow + t] = in ? to_f(cm[(t0 + t) * a.c_strides[1] + n]) : 0.f;
        }
        __syncthreads();

        F2 ddt2[kTokens], du[kTokens], y[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) ddt2[i] = du[i] = y[i] = {};
        const F2 total_dt = pack2(sum_dt.x, sum_dt.y);
        const float* hp = a.checkpoints + (checkpoint0 + t0 / kScanCheckpoint) * N * a.channels + c;
        if (k > 0 && lane < kTokens) {  // the next chunk's rows (the tokens before) into L2
            const int t = tw - kChunk + lane;
            prefetch_l2(x + t * a.x_strides[1] - 2 * lane);
            prefetch_l2(dtp + t * a.dt_strides[1] - 2 * lane);
            prefetch_l2(dout + static_cast<long long>(t) * a.channels - 2 * lane);
            if (GATED) prefetch_l2(z + t * a.z_strides[1] - 2 * lane);
        }
        Pack<float, 2> h_start;
        load_raw<VECTOR, false>(h_start, hp, pn);  // the state that the chunk starts from, a column ahead
        for (int n = 0; n < N; ++n) {
            const int buf = n & 1;
            const F2 a2 = *reinterpret_cast<const F2*>(sa + n * kBwdChannels + 2 * lane);
            F2 hs = pack2(h_start.v[0], h_start.v[1]);
            if (n + 1 < N) load_raw<VECTOR, false>(h_start, hp + static_cast<long long>(n + 1) * a.channels, pn);
            float bt[kTokens], ct[kTokens];
#pragma unroll
            for (int i = 0; i < kTokens; i += 4) {
                *reinterpret_cast<float4*>(bt + i) = *reinterpret_cast<const float4*>(sb + n * kRow + w * kTokens + i);
                *reinterpret_cast<float4*>(ct + i) = *reinterpret_cast<const float4*>(sc + n * kRow + w * kTokens + i);
            }
            F2 al[kTokens], h[kTokens];
            F2 end_h = {}, end_g = {};
#pragma unroll
            for (int i = 0; i < kTokens; ++i) {
                al[i] = exp2_2(mul2(dt[i], a2));
                h[i] = mul2(u[i], pack2(bt[i], bt[i]));
                end_h = fma2(al[i], end_h, h[i]);
            }
#pragma unroll
            for (int i = kTokens - 1; i >= 0; --i) end_g = mul2(al[i], fma2(pack2(ct[i], ct[i]), dy[i], end_g));
            {
                const float2 p = unpack2(exp2_2(mul2(total_dt, a2))), e = unpack2(end_h);
                ex_h[(buf * kWarps + w) * 32 + lane] = make_float4(p.x, p.y, e.x, e.y);
                ex_g[(buf * kWarps + w) * 32 + lane] = unpack2(end_g);
            }
            __syncthreads();
            // dA of the column before, left by all warps before this barrier: one of them adds it up
            if (n > 0 && w == ((n - 1) & (kWarps - 1))) {
                float2* at = reinterpret_cast<float2*>(sda + (n - 1) * kBwdChannels + 2 * lane);
                float2 sum = *at;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) {
                    const float2 d = ex_a[((buf ^ 1) * kWarps + v) * 32 + lane];
                    sum = make_float2(sum.x + d.x, sum.y + d.y);
                }
                *at = sum;
            }
            // all of them loaded at once; whether a warp lies before or behind is the same for all lanes
            F2 gs = *reinterpret_cast<const F2*>(sg + (side * N + n) * kBwdChannels + 2 * lane);
            F2 decay[kWarps], end[kWarps];
#pragma unroll
            for (int v = 0; v < kWarps; ++v) {
                const F2* before = reinterpret_cast<const F2*>(ex_h + (buf * kWarps + v) * 32 + lane);
                const F2* behind = reinterpret_cast<const F2*>(ex_g + (buf * kWarps + v) * 32 + lane);
                decay[v] = *before;
                end[v] = v < w ? before[1] : *behind;
            }
#pragma unroll
            for (int v = 0; v < kWarps - 1; ++v)
                if (v < w) hs = fma2(decay[v], hs, end[v]);
#pragma unroll
            for (int v = kWarps - 1; v > 0; --v)
                if (v > w) gs = fma2(decay[v], gs, end[v]);
            if (w == 0) {
                *reinterpret_cast<F2*>(sg + ((side ^ 1) * N + n) * kBwdChannels + 2 * lane) = fma2(decay[0], gs, end_g);
            }
            float v16[16];  // dB, dC of the tokens, over this lane's channels
            {
                F2 prev = hs;
#pragma unroll
                for (int i = 0; i < kTokens; ++i) {
                    prev = fma2(al[i], prev, h[i]);
                    h[i] = prev;
                    v16[8 + i] = sum2(mul2(dy[i], prev));
                    if (GATED) y[i] = fma2(pack2(ct[i], ct[i]), prev, y[i]);
                }
            }
            F2 da = {};
#pragma unroll
            for (int i = kTokens - 1; i >= 0; --i) {
                const F2 gt = fma2(pack2(ct[i], ct[i]), dy[i], gs);
                v16[i] = sum2(mul2(gt, u[i]));
                du[i] = fma2(gt, pack2(bt[i], bt[i]), du[i]);
                gs = mul2(gt, al[i]);
                const F2 q = mul2(gs, i > 0 ? h[i > 0 ? i - 1 : 0] : hs);
                ddt2[i] = fma2(q, a2, ddt2[i]);
                da = fma2(q, dt[i], da);
            }
            ex_a[(buf * kWarps + w) * 32 + lane] = unpack2(da);
            const float r = sum_lanes16(v16, lane);
            // value lane / 2: dB of tokens 0..7, then dC; this warp alone reads these places
            if ((lane & 1) == 0) (lane < 16 ? sb : sc)[n * kRow + w * kTokens + ((lane >> 1) & 7)] = r;
        }
        __syncthreads();
        if (w == ((N - 1) & (kWarps - 1))) {
            float2* at = reinterpret_cast<float2*>(sda + (N - 1) * kBwdChannels + 2 * lane);
            float2 sum = *at;
#pragma unroll
            for (int v = 0; v < kWarps; ++v) {
                const float2 d = ex_a[(((N - 1) & 1) * kWarps + v) * 32 + lane];
                sum = make_float2(sum.x + d.x, sum.y + d.y);
            }
            *at = sum;
        }
        for (int i = tid; i < N * kChunk; i += 32 * kWarps) {
            const int t = i / N, n = i % N;
            if (t0 + t < s.t1) {
                const long long at = static_cast<long long>(t0 + t) * a.groups * N + n;
                db[at] = sb[n * kRow + t];
                dc[at] = sc[n * kRow + t];
            }
        }
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int t = tw + i, n = t < s.t1 ? pn : 0;
            load_raw<VECTOR, false>(xr[i], x + t * a.x_strides[1], n);
            load_raw<VECTOR, false>(dr[i], dtp + t * a.dt_strides[1], n);
            if (GATED) {
                load_raw<VECTOR, false>(zr[i], z + t * a.z_strides[1], n);
                load_raw<VECTOR, false>(gr[i], dout + static_cast<long long>(t) * a.channels, n);
            }
        }
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int t = tw + i, n = t < s.t1 ? pn : 0;
            const float2 xv = pair_f(xr[i]);
            const float2 dv = unpack2(dt[i]), duv = unpack2(du[i]), dyv = unpack2(dy[i]), qa = unpack2(ddt2[i]);
            constexpr float kLn2 = 0.6931471805599453f;
            float2 dd = make_float2(fmaf(qa.x, kLn2, xv.x * duv.x), fmaf(qa.y, kLn2, xv.y * duv.y));
            if (a.softplus) {
                const float2 raw = pair_f(dr[i]);
                dd.x *= sigmoid_fast(raw.x + bias.x);
                dd.y *= sigmoid_fast(raw.y + bias.y);
            }
            const long long at = (first_token + t) * a.channels + c;
            store_pair<VECTOR>(static_cast<T*>(g.dx) + at,
                               make_float2(fmaf(dv.x, duv.x, skip.x * dyv.x), fmaf(dv.y, duv.y, skip.y * dyv.y)), n);
            store_pair<VECTOR>(static_cast<T*>(g.ddt) + at, dd, n);
            if (GATED) {
                const float2 zv = pair_f(zr[i]), yv = unpack2(y[i]), o = pair_f(gr[i]);
                const float gx = sigmoid_fast(zv.x), gy = sigmoid_fast(zv.y);
                store_pair<VECTOR>(static_cast<T*>(g.dz) + at,
                                   make_float2(o.x * fmaf(skip.x, xv.x, yv.x) * gx * fmaf(zv.x, 1.f - gx, 1.f),
                                               o.y * fmaf(skip.y, xv.y, yv.y) * gy * fmaf(zv.y, 1.f - gy, 1.f)), n);
            }
            if (n > 0) {
                dskip = make_float2(fmaf(dyv.x, xv.x, dskip.x), fmaf(dyv.y, xv.y, dskip.y));
                dbias = make_float2(dbias.x + dd.x, dbias.y + dd.y);
            }
        }
        side ^= 1;
        __syncthreads();  // before B and C of the next chunk
    }

    // ---- parameters: this item's row of the table, and the gradient of the initial state
    float2* ex = reinterpret_cast<float2*>(ex_h);
    ex[w * 32 + lane] = dskip;
    ex[(kWarps + w) * 32 + lane] = dbias;
    __syncthreads();
    float* row = l.channel_part + item * (N + 2) * a.channels + cb.first;
    for (int i = tid; i < (N + 2) * kBwdChannels; i += 32 * kWarps) {
        const int n = i / kBwdChannels, ch = i % kBwdChannels;
        if (ch >= cb.n) continue;
        float v = 0.f;
        if (n < N) {
            v = sda[i];
        } else {
            const float* part = reinterpret_cast<const float*>(ex + (n == N ? 0 : kWarps) * 32);
            for (int k = 0; k < kWarps; ++k) v += part[k * kBwdChannels + ch];
        }
        row[static_cast<long long>(n) * a.channels + ch] = v;
        if (n < N && s.first && g.dinitial != nullptr)
            g.dinitial[(static_cast<long long>(s.seq) * a.channels + cb.first + ch) * N + n] =
                sg[(side * N + n) * kBwdChannels + ch];
    }
}

// dB, dC: the tables of the blocks of channels of a group, added up in their order.
template <class T>
__global__ void __launch_bounds__(256)
scan_shared_sum_kernel(const float* part, int tables, long long count, T* db, T* dc) {
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= 2 * count) return;
    const bool second = i >= count;
    const float* src = part + (second ? tables * count + (i - count) : i);
    float sum = 0.f;
#pragma unroll 8
    for (int k = 0; k < tables; ++k) sum += src[k * count];
    (second ? dc : db)[second ? i - count : i] = from_f<T>(sum);
}

// dA, dD, d_dt_bias: the items' rows, added up in their order.
__global__ void __launch_bounds__(kSumCols * kSumRows)
scan_channel_sum_kernel(const float* table, long long rows, int channels, int dstate, float* dA, float* dD, float* dbias) {
    column_sums(table, rows, static_cast<long long>(channels) * (dstate + 2), [&](long long col, float v) {
        const int n = static_cast<int>(col / channels), c = static_cast<int>(col - static_cast<long long>(n) * channels);
        if (n < dstate)
            dA[static_cast<long long>(c) * dstate + n] = v;
        else if (n == dstate && dD != nullptr)
            dD[c] = v;
        else if (n > dstate && dbias != nullptr)
            dbias[c] = v;
    });
}

struct BwdSizes {
    ScanSegments segments;
    ScanBlocks blocks;
    size_t ends, shared, channel;  // floats
    long long all_tokens;
};
BwdSizes bwd_sizes(const SsdScanArgs& a) {
    BwdSizes z;
    z.segments = scan_segments(a, kBwdChannels, sm_count());
    z.blocks = scan_blocks(a.channels, a.groups, kBwdChannels);
    z.all_tokens = a.cu_seqlens ? a.tokens : a.tokens * a.rows;
    z.ends = scan_segment_floats(a, z.segments);
    z.shared = 2 * static_cast<size_t>(z.blocks.per_group) * z.all_tokens * a.groups * a.dstate;
    z.channel = static_cast<size_t>(z.segments.items) * (a.dstate + 2) * a.channels;
    return z;
}

}  // namespace

}  // namespace ssd

extern "C" size_t ssd_selective_scan_grad_work_bytes(const SsdScanArgs* args) {
    using namespace ssd;
    if (args == nullptr || scan_check(*args) != SSD_OK) return 0;
    const BwdSizes z = bwd_sizes(*args);
    return sizeof(float) * (z.ends + z.shared + z.channel);
}

extern "C" int ssd_selective_scan_bwd(const SsdScanGradArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdScanGradArgs& g = *args;
    const SsdScanArgs& a = g.forward;
    if (const int rc = scan_check(a); rc != SSD_OK) return rc;
    if (!g.work || !g.dA || (a.tokens > 0 && (!a.checkpoints || !g.dout || !g.dx || !g.ddt || !g.dbm || !g.dcm || (a.z && !g.dz))))
        return SSD_ERR_NULL;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const BwdSizes z = bwd_sizes(a);
    if (z.segments.split)
        if (const int rc = scan_segment_states(a, z.segments, g.work, g.dout, g.dfinal, st); rc != SSD_OK) return rc;
    const BwdLaunch l{scan_map(a, z.segments.span), z.blocks, z.segments.split, g.work, g.work + z.ends,
                      g.work + z.ends + z.shared, z.all_tokens};
    const long long ctas = z.segments.items * z.blocks.count(a.groups);
    const long long cells = z.all_tokens * a.groups * a.dstate, grid = (2 * cells + 255) / 256;
    if (ctas > 0x7fffffffLL || grid > 0x7fffffffLL) return SSD_ERR_RANGE;
    const int rc = with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const bool pairs = scan_pairs(a, sizeof(T)) && aligned_to(2 * sizeof(T), g.dout, g.dx, g.ddt, g.dz);
        const auto launch = [&](auto kernel) {
            static std::atomic<uint64_t> done[4];
            if (const int e = set_max_smem_once(reinterpret_cast<const void*>(kernel), bwd_smem(kScanMaxState),
                                                done[2 * pairs + (a.z != nullptr)]);
                e != SSD_OK)
                return e;
            launch_plain(kernel, static_cast<unsigned>(ctas), 32 * kWarps, bwd_smem(a.dstate), st, g, l);
            return launch_status();
        };
        const int e = a.z ? (pairs ? launch(selective_bwd_kernel<T, true, true>) : launch(selective_bwd_kernel<T, false, true>))
                          : (pairs ? launch(selective_bwd_kernel<T, true, false>) : launch(selective_bwd_kernel<T, false, false>));
        if (e != SSD_OK || cells == 0) return e;
        launch_plain(scan_shared_sum_kernel<T>, static_cast<unsigned>(grid), 256, 0, st, l.shared_part, z.blocks.per_group, cells,
                     static_cast<T*>(g.dbm), static_cast<T*>(g.dcm));
        return launch_status();
    });
    if (rc != SSD_OK) return rc;
    const long long cols = static_cast<long long>(a.channels) * (a.dstate + 2);
    launch_plain(scan_channel_sum_kernel, static_cast<unsigned>((cols + kSumCols - 1) / kSumCols), kSumCols * kSumRows, 0, st,
                 l.channel_part, z.segments.items, a.channels, a.dstate, g.dA, g.dD, g.d_dt_bias);
    return launch_status();
}
