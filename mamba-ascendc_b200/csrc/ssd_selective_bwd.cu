// Selective scan, gradients.  With dy = dout silu(z) and g the gradient of the states,
//
//   g_t = C_t dy_t + a_{t+1} g_{t+1} ;  dC_t[n] = sum_c dy_t h_t[n] ;  dB_t[n] = sum_c g_t[n] dt_t x_t ;  du_t = sum_n g_t[n] B_t[n]
//   q_t[n] = g_t[n] a_t[n] h_{t-1}[n] ;  ddt_t = x_t du_t + sum_n q_t[n] A[n] ;  dA[n] = sum_t q_t[n] dt_t ;  dx_t = dt_t du_t + D dy_t
//
// What bounds it: instructions, 35 for each (token, channel, state column) as counted: 16 are the arithmetic, the others the sums
// of dB and dC over the channels, which lie along the lanes, the exchange between the warps of a chunk, and what each (token,
// channel) takes.  The bytes are few beside that.
//
// Layout: a lane owns two neighbouring channels, a warp kTokens tokens of 64 channels, a CTA a chunk of kWarps * kTokens tokens,
// which it walks from the sequence's end.  For one state column at a time each warp forms its exponentials once, runs the
// recurrences of h and g from zero over its tokens, and puts their ends and the product of its decays into shared memory;
// after one barrier it folds those of the warps before (behind) it into its true start, and runs both recurrences again on
// the exponentials it still holds.  h enters a chunk from the forward pass's checkpoints, g from the chunk behind.  Sums over
// n stay with the thread; sums over the lanes go through shared memory, 38 instructions for 16 values against 62 with shuffles.
// dB and dC replace B and C in shared memory (a warp's tokens are its own) and leave as one table per block of channels, summed
// in a fixed order by scan_shared_sum_kernel.
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

constexpr int kValues = 2 * kTokens;  // dB and dC of a warp's tokens
constexpr int kLaneRow = 32 + 4;      // a value of all lanes, padded so that eight lanes read sixteen of them without conflict
size_t bwd_smem(int dstate) {
    return sizeof(float) * (2 * dstate * kRow + 3 * dstate * kBwdChannels + 2 * kWarps * 32 * (4 + 4 + 2) + kWarps * kValues * kLaneRow);
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Sums over the 32 lanes of 16 values each: lane l returns that of value l / 2.  `rows` is the warp's own.
__device__ __forceinline__ float sum_lanes(const float (&v)[kValues], float* rows, int lane) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kValues; ++j) rows[j * kLaneRow + lane] = v[j];
    __syncwarp();
    const float4* half = reinterpret_cast<const float4*>(rows + (lane >> 1) * kLaneRow + (lane & 1) * 16);
    float4 sum = half[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const float4 q = half[i];
        sum = make_float4(sum.x + q.x, sum.y + q.y, sum.z + q.z, sum.w + q.w);
    }
    const float mine = (sum.x + sum.y) + (sum.z + sum.w);
    return mine + __shfl_xor_sync(0xffffffffu, mine, 1);
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
    float2* sa = reinterpret_cast<float2*>(sc + N * kRow);  // [N][32] A log2(e) of the lane's channels
    float2* sg = sa + N * 32;                       // [N][32] gradient of the state behind the chunk
    float2* sda = sg + N * 32;                      // [N][32] dA
    float4* ex_h = reinterpret_cast<float4*>(sda + N * 32);  // [2][warps][32] decay, end of h
    float4* ex_g = ex_h + 2 * kWarps * 32;                   // [2][warps][32] decay, end of g
    float2* ex_a = reinterpret_cast<float2*>(ex_g + 2 * kWarps * 32);  // [2][warps][32] dA of the warp
    float* rows = reinterpret_cast<float*>(ex_a + 2 * kWarps * 32) + w * kValues * kLaneRow;

    const int c = cb.first + 2 * lane, pn = max(min(cb.n - 2 * lane, 2), 0);
    for (int i = tid; i < N * kBwdChannels; i += 32 * kWarps) {
        const int n = i / kBwdChannels, ch = i % kBwdChannels;
        const bool in = ch < cb.n;
        float end = 0.f;
        if (in) {
            if (l.split)
                end = l.ends[(item * N + n) * a.channels + cb.first + ch];
            else if (g.dfinal != nullptr)
                end = g.dfinal[(static_cast<long long>(s.seq) * a.channels + cb.first + ch) * N + n];
        }
        reinterpret_cast<float*>(sa)[i] = in ? decay_rate(a.A[static_cast<long long>(cb.first + ch) * N + n]) : 0.f;
        reinterpret_cast<float*>(sda)[i] = 0.f;
        reinterpret_cast<float*>(sg)[i] = end;
    }
    float2 bias = make_float2(0.f, 0.f), skip = bias, dskip = bias, dbias = bias;
    if (a.dt_bias != nullptr) bias = make_float2(pn > 0 ? a.dt_bias[c] : 0.f, pn > 1 ? a.dt_bias[c + 1] : 0.f);
    if (a.D != nullptr) skip = make_float2(pn > 0 ? a.D[c] : 0.f, pn > 1 ? a.D[c + 1] : 0.f);

    const Rows<T> xs(static_cast<const T*>(a.x) + first_row(l.map, s, a.x_strides) + c, a.x_strides[1]);
    const Rows<T> dts(static_cast<const T*>(a.dt) + first_row(l.map, s, a.dt_strides) + c, a.dt_strides[1]);
    const Rows<T> zs(static_cast<const T*>(a.z) + first_row(l.map, s, a.z_strides) + c, a.z_strides[1]);
    const Rows<T> douts(static_cast<const T*>(g.dout) + first_token * a.channels + c, a.channels);
    const Rows<T> bs(static_cast<const T*>(a.bm) + first_row(l.map, s, a.b_strides) + cb.group * a.b_strides[2], a.b_strides[1]);
    const Rows<T> cs(static_cast<const T*>(a.cm) + first_row(l.map, s, a.c_strides) + cb.group * a.c_strides[2], a.c_strides[1]);
    const Rows<float> dbs(db, a.groups * N), dcs(dc, a.groups * N);
    const long long out0 = first_token * a.channels + c;
    const Rows<T> dxs(static_cast<T*>(g.dx) + out0, a.channels), ddts(static_cast<T*>(g.ddt) + out0, a.channels);
    const Rows<T> dzs(static_cast<T*>(g.dz) + out0, a.channels);
    const long long checkpoint0 = l.map.cu == nullptr
                                      ? s.seq * ((l.map.tokens + kScanCheckpoint - 1) / kScanCheckpoint)
                                      : s.origin / kScanCheckpoint + s.seq;
    // B and C of a chunk: a thread has a token and every fourth quad of columns
    const int quad_t = tid % kChunk, quads = (N + 3) / 4;

    const int chunks = (s.t1 - s.t0 + kChunk - 1) / kChunk;
    for (int k = chunks - 1; k >= 0; --k) {
        const int t0 = s.t0 + k * kChunk, tw = t0 + w * kTokens;
        // ---- this warp's tokens
        F2 dt[kTokens], u[kTokens], dy[kTokens];
        float2 sum_dt = make_float2(0.f, 0.f);
        Pack<T, 2> xr[kTokens], dr[kTokens], zr[kTokens], gr[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int t = tw + i, n = t < s.t1 ? pn : 0;
            load_raw<VECTOR, false>(xr[i], xs.at(t), n);
            load_raw<VECTOR, false>(dr[i], dts.at(t), n);
            load_raw<VECTOR, false>(gr[i], douts.at(t), n);
            if (GATED) load_raw<VECTOR, false>(zr[i], zs.at(t), n);
        }
        for (int q = tid / kChunk; q < quads; q += 32 * kWarps / kChunk) {
            const int n = q * 4, in = t0 + quad_t < s.t1 ? min(N - n, 4) : 0;
            Pack<T, 4> br, cr;
            load_raw<VECTOR, false>(br, bs.at(t0 + quad_t) + n, in);
            load_raw<VECTOR, false>(cr, cs.at(t0 + quad_t) + n, in);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (VECTOR || n + j < N) {
                    sb[(n + j) * kRow + quad_t] = to_f(br.v[j]);
                    sc[(n + j) * kRow + quad_t] = to_f(cr.v[j]);
                }
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
        __syncthreads();

        F2 ddt2[kTokens], du[kTokens], y[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) ddt2[i] = du[i] = y[i] = {};
        const float* hp = a.checkpoints + (checkpoint0 + t0 / kScanCheckpoint) * N * a.channels + c;
        if (k > 0 && lane < kTokens) {  // the next chunk's rows (the tokens before) into L2
            const int t = tw - kChunk + lane;
            prefetch_l2(xs.at(t) - 2 * lane);
            prefetch_l2(dts.at(t) - 2 * lane);
            prefetch_l2(douts.at(t) - 2 * lane);
            if (GATED) prefetch_l2(zs.at(t) - 2 * lane);
        }
        Pack<float, 2> h_start;  // the state that the chunk starts from, a column ahead
        load_raw<VECTOR, false>(h_start, hp, pn);
        // of the column: A, g behind the chunk, dA, and this warp's tokens of B and C; and this parity's exchange
        const float2* an = sa + lane;
        float2* gn = sg + lane;
        float2* dan = sda + lane;
        float* bn = sb + w * kTokens;
        const int c_off = N * kRow;
        float4* eh = ex_h + lane;
        float2* ea = ex_a + lane;
        constexpr int to_h_g = 2 * kWarps * 32;
        float2 g_before = make_float2(0.f, 0.f);  // warp 0: gradient of the state before the chunk, of the last column
        for (int n = 0; n < N; ++n) {
            const float2 a2 = *an;
            F2 hs = pack2(h_start.v[0], h_start.v[1]);
            hp += a.channels;
            if (n + 1 < N) load_raw<VECTOR, false>(h_start, hp, pn);
            float bt[kTokens], ct[kTokens];
#pragma unroll
            for (int i = 0; i < kTokens; i += 4) {
                *reinterpret_cast<float4*>(bt + i) = *reinterpret_cast<const float4*>(bn + i);
                *reinterpret_cast<float4*>(ct + i) = *reinterpret_cast<const float4*>(bn + c_off + i);
            }
            F2 al[kTokens], h[kTokens];
            F2 end_h = {}, end_g = {};
#pragma unroll
            for (int i = 0; i < kTokens; ++i) {
                al[i] = pack2(decay(dt[i].x, a2.x), decay(dt[i].y, a2.y));
                h[i] = pack2(u[i].x * bt[i], u[i].y * bt[i]);
                end_h = fma2(al[i], end_h, h[i]);
            }
#pragma unroll
            for (int i = kTokens - 1; i >= 0; --i)
                end_g = pack2(al[i].x * fmaf(ct[i], dy[i].x, end_g.x), al[i].y * fmaf(ct[i], dy[i].y, end_g.y));
            {
                const float px = decay(sum_dt.x, a2.x), py = decay(sum_dt.y, a2.y);
                eh[w * 32] = make_float4(px, py, end_h.x, end_h.y);
                eh[to_h_g + w * 32] = make_float4(px, py, end_g.x, end_g.y);
            }
            __syncthreads();
            // what all warps left of the column before: one of them adds up its dA, warp 0 moves its g on
            if (n > 0) {
                if (w == ((n - 1) & (kWarps - 1))) {
                    float2 sum = dan[-32];
                    const float2* last = ex_a + lane + (((n - 1) & 1) ? kWarps * 32 : 0);
#pragma unroll
                    for (int v = 0; v < kWarps; ++v) sum = make_float2(sum.x + last[v * 32].x, sum.y + last[v * 32].y);
                    dan[-32] = sum;
                }
                if (w == 0) gn[-32] = g_before;
            }
            // all loaded at once; whether a warp lies before or behind is the same for all lanes
            F2 gs = pack2(gn->x, gn->y);
            float4 e[kWarps];
#pragma unroll
            for (int v = 0; v < kWarps; ++v)
                e[v] = eh[(v < w ? 0 : to_h_g) + v * 32];
#pragma unroll
            for (int v = 0; v < kWarps - 1; ++v)
                if (v < w) hs = pack2(fmaf(e[v].x, hs.x, e[v].z), fmaf(e[v].y, hs.y, e[v].w));
#pragma unroll
            for (int v = kWarps - 1; v > 0; --v)
                if (v > w) gs = pack2(fmaf(e[v].x, gs.x, e[v].z), fmaf(e[v].y, gs.y, e[v].w));
            float v16[kValues];  // dB, dC of the tokens, over this lane's channels
            {
                F2 prev = hs;
#pragma unroll
                for (int i = 0; i < kTokens; ++i) {
                    prev = fma2(al[i], prev, h[i]);
                    h[i] = prev;
                    v16[kTokens + i] = fmaf(dy[i].y, prev.y, dy[i].x * prev.x);
                    if (GATED) y[i] = pack2(fmaf(ct[i], prev.x, y[i].x), fmaf(ct[i], prev.y, y[i].y));
                }
            }
            F2 da = {};
#pragma unroll
            for (int i = kTokens - 1; i >= 0; --i) {
                const F2 gt = pack2(fmaf(ct[i], dy[i].x, gs.x), fmaf(ct[i], dy[i].y, gs.y));
                v16[i] = fmaf(gt.y, u[i].y, gt.x * u[i].x);
                du[i] = pack2(fmaf(gt.x, bt[i], du[i].x), fmaf(gt.y, bt[i], du[i].y));
                gs = mul2(gt, al[i]);
                const F2 q = mul2(gs, i > 0 ? h[i > 0 ? i - 1 : 0] : hs);
                ddt2[i] = pack2(fmaf(q.x, a2.x, ddt2[i].x), fmaf(q.y, a2.y, ddt2[i].y));
                da = fma2(q, dt[i], da);
            }
            g_before = make_float2(gs.x, gs.y);
            ea[w * 32] = make_float2(da.x, da.y);
            const float r = sum_lanes(v16, rows, lane);
            // value lane / 2: dB of tokens 0..7, then dC; this warp alone reads these places
            if ((lane & 1) == 0) bn[(lane < 16 ? 0 : c_off) + ((lane >> 1) & 7)] = r;
            an += 32;
            gn += 32;
            dan += 32;
            bn += kRow;
            // the other parity
            eh += n % 2 == 0 ? kWarps * 32 : -kWarps * 32;
            ea += n % 2 == 0 ? kWarps * 32 : -kWarps * 32;
        }
        // on their way under the sums of the last column and the stores of dB and dC
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int t = tw + i, n = t < s.t1 ? pn : 0;
            load_raw<VECTOR, false>(xr[i], xs.at(t), n);
            load_raw<VECTOR, false>(dr[i], dts.at(t), n);
            if (GATED) {
                load_raw<VECTOR, false>(zr[i], zs.at(t), n);
                load_raw<VECTOR, false>(gr[i], douts.at(t), n);
            }
        }
        __syncthreads();
        if (w == ((N - 1) & (kWarps - 1))) {
            float2 sum = dan[-32];
            const float2* last = ex_a + lane + (((N - 1) & 1) ? kWarps * 32 : 0);
#pragma unroll
            for (int v = 0; v < kWarps; ++v) sum = make_float2(sum.x + last[v * 32].x, sum.y + last[v * 32].y);
            dan[-32] = sum;
        }
        if (w == 0) gn[-32] = g_before;
        if (t0 + quad_t < s.t1) {
            for (int q = tid / kChunk; q < quads; q += 32 * kWarps / kChunk) {
                const int n = q * 4;
                float fb[4], fc[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (VECTOR || n + j < N) fb[j] = sb[(n + j) * kRow + quad_t], fc[j] = sc[(n + j) * kRow + quad_t];
                store_f<VECTOR>(dbs.to(t0 + quad_t) + n, fb, min(N - n, 4));
                store_f<VECTOR>(dcs.to(t0 + quad_t) + n, fc, min(N - n, 4));
            }
        }
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int t = tw + i, n = t < s.t1 ? pn : 0;
            const float2 xv = pair_f(xr[i]);
            constexpr float kLn2 = 0.6931471805599453f;
            float2 dd = make_float2(fmaf(ddt2[i].x, kLn2, xv.x * du[i].x), fmaf(ddt2[i].y, kLn2, xv.y * du[i].y));
            if (a.softplus) {
                const float2 raw = pair_f(dr[i]);
                dd.x *= sigmoid_fast(raw.x + bias.x);
                dd.y *= sigmoid_fast(raw.y + bias.y);
            }
            store_pair<VECTOR>(dxs.to(t), make_float2(fmaf(dt[i].x, du[i].x, skip.x * dy[i].x), fmaf(dt[i].y, du[i].y, skip.y * dy[i].y)),
                               n);
            store_pair<VECTOR>(ddts.to(t), dd, n);
            if (GATED) {
                const float2 zv = pair_f(zr[i]), o = pair_f(gr[i]);
                const float gx = sigmoid_fast(zv.x), gy = sigmoid_fast(zv.y);
                store_pair<VECTOR>(dzs.to(t), make_float2(o.x * fmaf(skip.x, xv.x, y[i].x) * gx * fmaf(zv.x, 1.f - gx, 1.f),
                                                          o.y * fmaf(skip.y, xv.y, y[i].y) * gy * fmaf(zv.y, 1.f - gy, 1.f)), n);
            }
            if (n > 0) {
                dskip = make_float2(fmaf(dy[i].x, xv.x, dskip.x), fmaf(dy[i].y, xv.y, dskip.y));
                dbias = make_float2(dbias.x + dd.x, dbias.y + dd.y);
            }
        }
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
            v = reinterpret_cast<const float*>(sda)[i];
        } else {
            const float* part = reinterpret_cast<const float*>(ex + (n == N ? 0 : kWarps) * 32);
            for (int k = 0; k < kWarps; ++k) v += part[k * kBwdChannels + ch];
        }
        row[static_cast<long long>(n) * a.channels + ch] = v;
        if (n < N && s.first && g.dinitial != nullptr)
            g.dinitial[(static_cast<long long>(s.seq) * a.channels + cb.first + ch) * N + n] =
                reinterpret_cast<const float*>(sg)[i];
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
    z.ends = (scan_segment_floats(a, z.segments) + 3) / 4 * 4;  // the tables behind are written four floats at a time
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
