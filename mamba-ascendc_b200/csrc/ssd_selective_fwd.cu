// Selective scan, forward, and the segment states that both directions take:
//
//   a_t[n] = exp(dt_t A[n]) ;  h_t[n] = a_t[n] h_{t-1}[n] + dt_t x_t B_t[n] ;  y_t = sum_n C_t[n] h_t[n]   for every channel
//
// What bounds it: one exponential and two multiply-adds with two products for each (token, channel, state column), not the
// bytes (with 16 columns 16 exponentials for 8 bytes).  An SM forms 16 exponentials a cycle, eight cycles for a warp's.
// The walk over the tokens is serial with the state in registers, so that each exponential is formed once.
//
// Layout: a lane owns a channel, a warp NPL state columns of 32 channels, NW warps all columns of them, a CTA `cg` such sets.
// B and C are the same for all lanes (one broadcast load for four columns), and nothing is exchanged between lanes; the NW
// partial sums of y meet in shared memory.  Tokens pass through shared memory kScanTile at a time: dt (softplus taken once)
// and dt x as pairs, B and C in fp32.  The next tile's loads are in flight under the walk.
//
// kMode: the forward pass itself; each segment's end state from a zero start; or backward in time, the gradient that a segment
// hands to the state before it, e <- a_t (e + C_t dy_t), with dy = dout silu(z).
#include <type_traits>

#include "ssd_selective.cuh"

namespace ssd {

namespace {

constexpr int kScanTile = 32;
enum ScanMode { kForward, kEndState, kStartGradient };

struct ScanLaunch {
    SeqMap map;
    ScanBlocks blocks;
    int cg;
    bool split;            // start states come from `work`
    float* work;           // [items][dstate][channels], [items][channels]
    const void* dout;      // kStartGradient
};

template <class T, int NPL, int NW, bool VECTOR, ScanMode kMode>
__global__ void __launch_bounds__(32 * NW * (NW >= 8 ? 1 : 8 / NW))
selective_walk_kernel(const SsdScanArgs a, const ScanLaunch l) {
    constexpr int kCols = NPL * NW;               // state columns, those behind dstate are zeros
    constexpr int kPairs = kScanTile / (2 * NW);  // channel pairs of a tile that a thread stages
    constexpr int kShared = 2 * NPL;              // B and C elements that a thread stages (with one channel set)
    constexpr bool kReverse = kMode == kStartGradient;
    extern __shared__ __align__(16) float walk_smem[];
    const int blocks = l.blocks.count(a.groups);
    const long long item = blockIdx.x / blocks;
    const ChannelBlock cb = channel_block(l.blocks, blockIdx.x % blocks, a.channels, a.groups);
    Span s;
    if (!locate(l.map, item, s)) return;
    const int tid = threadIdx.x, threads = 32 * NW * l.cg, lane = tid & 31, warp = tid >> 5;
    const int channels_here = 32 * l.cg, row_pairs = 16 * l.cg;  // a power of two
    const long long rows_before = l.map.cu == nullptr ? s.seq * l.map.tokens : 0;

    if (s.pad) {
        if (kMode == kForward)
            for (long long i = tid; i < static_cast<long long>(s.t1 - s.t0) * cb.n; i += threads) {
                const long long t = i / cb.n;
                static_cast<T*>(a.out)[(s.origin + s.t0 + t) * a.channels + cb.first + i % cb.n] = from_f<T>(0.f);
            }
        return;
    }

    float2* sdu = reinterpret_cast<float2*>(walk_smem);       // [tile][channels] dt, dt x (or dy)
    float* sb = walk_smem + 2 * kScanTile * channels_here;    // [tile][kCols] B (or C)
    float* sc = sb + kScanTile * kCols;                       // [tile][kCols]
    float* sy = sc + kScanTile * kCols;                       // [NW][tile][channels]

    // ---- the walk's own state
    const int wn = warp % NW, wc = warp / NW;
    const int mine = wc * 32 + lane, c = cb.first + mine, n0 = wn * NPL;
    const bool live = mine < cb.n;
    F2 h[NPL / 2], a2[NPL / 2];
    float sum_dt = 0.f;
    const float* start = l.work + item * a.dstate * a.channels;
#pragma unroll
    for (int j = 0; j < NPL; j += 2) {
        float av[2], hv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = n0 + j + i;
            const bool in = live && n < a.dstate;
            av[i] = in ? a.A[static_cast<long long>(c) * a.dstate + n] * kLog2e : 0.f;
            hv[i] = 0.f;
            if (kMode == kForward && in) {
                if (l.split)
                    hv[i] = start[static_cast<long long>(n) * a.channels + c];
                else if (a.initial_state != nullptr)
                    hv[i] = a.initial_state[(static_cast<long long>(s.seq) * a.channels + c) * a.dstate + n];
            }
        }
        a2[j / 2] = pack2(av[0], av[1]);
        h[j / 2] = pack2(hv[0], hv[1]);
    }

    // ---- staging
    const T* x = static_cast<const T*>(a.x) + token_row(l.map, s, a.x_strides[0], a.x_strides[1], 0) + cb.first;
    const T* dt = static_cast<const T*>(a.dt) + token_row(l.map, s, a.dt_strides[0], a.dt_strides[1], 0) + cb.first;
    const T* z = static_cast<const T*>(a.z) + token_row(l.map, s, a.z_strides[0], a.z_strides[1], 0) + cb.first;
    const T* bm = static_cast<const T*>(kReverse ? a.cm : a.bm) +
                  token_row(l.map, s, kReverse ? a.c_strides[0] : a.b_strides[0], kReverse ? a.c_strides[1] : a.b_strides[1], 0) +
                  cb.group * (kReverse ? a.c_strides[2] : a.b_strides[2]);
    const int64_t b_step = kReverse ? a.c_strides[1] : a.b_strides[1];
    const T* cm = static_cast<const T*>(a.cm) + token_row(l.map, s, a.c_strides[0], a.c_strides[1], 0) +
                  cb.group * a.c_strides[2];
    T* out = static_cast<T*>(a.out) + (rows_before + s.origin) * a.channels + cb.first;
    const T* dout = static_cast<const T*>(l.dout) + (rows_before + s.origin) * a.channels + cb.first;
    const int pair = tid & (row_pairs - 1), first_row = tid / row_pairs, row_step = threads / row_pairs;  // 2 NW rows a step
    const int pn = min(cb.n - 2 * pair, 2);
    float2 bias = make_float2(0.f, 0.f), skip = bias;
    if (pn > 0) {
        if (a.dt_bias != nullptr)
            bias = make_float2(a.dt_bias[cb.first + 2 * pair], pn > 1 ? a.dt_bias[cb.first + 2 * pair + 1] : 0.f);
        if (a.D != nullptr) skip = make_float2(a.D[cb.first + 2 * pair], pn > 1 ? a.D[cb.first + 2 * pair + 1] : 0.f);
    }
    const int shared_each = kShared / l.cg;  // of them
    Pack<T, 2> xr[kPairs], dr[kPairs], zr[kPairs];
    Pack<T, 1> br[kShared];
    auto request = [&](int t0) {
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
            const int t = t0 + first_row + p * row_step;
            const int n = t < s.t1 ? pn : 0;
            load_raw<VECTOR, false>(dr[p], dt + t * a.dt_strides[1] + 2 * pair, n);
            if (kReverse) {
                load_raw<VECTOR, false>(xr[p], dout + static_cast<long long>(t) * a.channels + 2 * pair, n);
                if (a.z != nullptr) load_raw<VECTOR, false>(zr[p], z + t * a.z_strides[1] + 2 * pair, n);
            } else {
                load_raw<VECTOR, false>(xr[p], x + t * a.x_strides[1] + 2 * pair, n);
            }
        }
#pragma unroll
        for (int p = 0; p < kShared; ++p) {
            const int i = tid + (p / 2) * threads, t = t0 + i / kCols, n = i % kCols;
            const int in = p < shared_each && n < a.dstate && t < s.t1 ? 1 : 0;
            if (p % 2 == 0)
                load_raw<true, false>(br[p], bm + t * b_step + n, in);
            else if (kMode == kForward)
                load_raw<true, false>(br[p], cm + t * a.c_strides[1] + n, in);
        }
    };
    const int tiles = (s.t1 - s.t0 + kScanTile - 1) / kScanTile;
    auto tile_start = [&](int k) { return s.t0 + (kReverse ? tiles - 1 - k : k) * kScanTile; };
    if (tiles > 0) request(tile_start(0));

    for (int k = 0; k < tiles; ++k) {
        const int t0 = tile_start(k), nt = min(s.t1 - t0, kScanTile);
        float2 held[kPairs];  // x, for the skip connection
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
            const int row = first_row + p * row_step;
            const bool in = row < nt;
            const float2 xv = pair_f(xr[p]);
            float2 d = pair_f(dr[p]);
            d = make_float2(d.x + bias.x, d.y + bias.y);
            if (a.softplus) d = make_float2(softplus_series(d.x), softplus_series(d.y));
            if (!in) d = make_float2(0.f, 0.f);  // behind the last token the state stays
            float2 u;
            if (kReverse) {
                u = xv;
                if (a.z != nullptr) {
                    const float2 zv = pair_f(zr[p]);
                    u = make_float2(u.x * zv.x * sigmoid_fast(zv.x), u.y * zv.y * sigmoid_fast(zv.y));
                }
            } else {
                u = make_float2(d.x * xv.x, d.y * xv.y);
            }
            held[p] = xv;
            *reinterpret_cast<float4*>(&sdu[row * channels_here + 2 * pair]) = make_float4(d.x, u.x, d.y, u.y);
        }
#pragma unroll
        for (int p = 0; p < kShared; ++p)
            if (p < shared_each && (p % 2 == 0 || kMode == kForward))
                (p % 2 == 0 ? sb : sc)[tid + (p / 2) * threads] = to_f(br[p].v[0]);
        __syncthreads();
        if (k + 1 < tiles) request(tile_start(k + 1));
        if (kMode == kForward && a.z != nullptr) {
#pragma unroll
            for (int p = 0; p < kPairs; ++p) {
                const int t = t0 + first_row + p * row_step;
                load_raw<VECTOR, false>(zr[p], z + t * a.z_strides[1] + 2 * pair, t < s.t1 ? pn : 0);
            }
        }
        if (kMode == kForward && a.checkpoints != nullptr && (t0 - s.t0) % kScanCheckpoint == 0 && live) {
            const long long at = (l.map.cu == nullptr ? s.seq * ((l.map.tokens + kScanCheckpoint - 1) / kScanCheckpoint)
                                                      : s.origin / kScanCheckpoint + s.seq) + t0 / kScanCheckpoint;
            float* dst = a.checkpoints + at * a.dstate * a.channels + c;
#pragma unroll
            for (int j = 0; j < NPL; ++j) {
                const float2 v = unpack2(h[j / 2]);
                if (n0 + j < a.dstate) dst[static_cast<long long>(n0 + j) * a.channels] = j % 2 ? v.y : v.x;
            }
        }
        // kGroup tokens at a time, the next ones' operands on their way: nothing but the states depends on the token before.
        // Rows behind the last token have dt = 0; groups of nothing else are left out.
        constexpr int kGroup = NPL <= 4 ? 4 : NPL <= 8 ? 2 : 1, kGroups = kScanTile / kGroup;
        struct Operands {
            float2 du[kGroup];
            ulonglong2 b[kGroup][NPL / 4], c[kGroup][NPL / 4];
        };
        const auto row_of = [](int i) { return kReverse ? kScanTile - 1 - i : i; };
        const auto fetch = [&](Operands& o, int group) {
#pragma unroll
            for (int i = 0; i < kGroup; ++i) {
                const int row = row_of(group * kGroup + i);
                o.du[i] = sdu[row * channels_here + mine];
#pragma unroll
                for (int j = 0; j < NPL / 4; ++j) {
                    o.b[i][j] = *reinterpret_cast<const ulonglong2*>(sb + row * kCols + n0 + 4 * j);
                    if (kMode == kForward) o.c[i][j] = *reinterpret_cast<const ulonglong2*>(sc + row * kCols + n0 + 4 * j);
                }
            }
        };
        Operands now, next;
        fetch(now, 0);
#pragma unroll
        for (int group = 0; group < kGroups; ++group) {
            if (!kReverse && group * kGroup >= nt) break;
            if (group + 1 < kGroups) fetch(next, group + 1);
            if (!kReverse || row_of(group * kGroup + kGroup - 1) < nt) {
                F2 e[kGroup][NPL / 2];
                float y[kGroup];
#pragma unroll
                for (int i = 0; i < kGroup; ++i)
#pragma unroll
                    for (int j = 0; j < NPL / 2; ++j) e[i][j] = exp2_2(mul2(pack2(now.du[i].x, now.du[i].x), a2[j]));
#pragma unroll
                for (int i = 0; i < kGroup; ++i) {
                    const F2 uu = pack2(now.du[i].y, now.du[i].y);
                    if (kMode != kForward) sum_dt += now.du[i].x;
                    F2 sum = 0;
#pragma unroll
                    for (int j = 0; j < NPL / 4; ++j) {
                        const ulonglong2 bv = now.b[i][j];
                        if (kReverse) {
                            h[2 * j] = mul2(e[i][2 * j], fma2(uu, bv.x, h[2 * j]));
                            h[2 * j + 1] = mul2(e[i][2 * j + 1], fma2(uu, bv.y, h[2 * j + 1]));
                        } else {
                            h[2 * j] = fma2(e[i][2 * j], h[2 * j], mul2(uu, bv.x));
                            h[2 * j + 1] = fma2(e[i][2 * j + 1], h[2 * j + 1], mul2(uu, bv.y));
                        }
                        if (kMode == kForward) {
                            sum = fma2(now.c[i][j].x, h[2 * j], sum);
                            sum = fma2(now.c[i][j].y, h[2 * j + 1], sum);
                        }
                    }
                    y[i] = sum2(sum);
                }
                if (kMode == kForward) {
#pragma unroll
                    for (int i = 0; i < kGroup; ++i)
                        sy[(wn * kScanTile + row_of(group * kGroup + i)) * channels_here + mine] = y[i];
                }
            }
            now = next;
        }
        __syncthreads();
        if (kMode == kForward) {
#pragma unroll
            for (int p = 0; p < kPairs; ++p) {
                const int row = first_row + p * row_step;
                if (row >= nt) continue;
                float2 y = make_float2(skip.x * held[p].x, skip.y * held[p].y);
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float2 v = *reinterpret_cast<const float2*>(&sy[(w * kScanTile + row) * channels_here + 2 * pair]);
                    y.x += v.x;
                    y.y += v.y;
                }
                if (a.z != nullptr) {
                    const float2 zv = pair_f(zr[p]);
                    y.x *= zv.x * sigmoid_fast(zv.x);
                    y.y *= zv.y * sigmoid_fast(zv.y);
                }
                store_pair<VECTOR>(out + static_cast<long long>(t0 + row) * a.channels + 2 * pair, y, pn);
            }
        }
    }
    if (!live) return;
    if (kMode == kForward) {
        if (!s.last || a.final_state == nullptr) return;
        float* dst = a.final_state + (static_cast<long long>(s.seq) * a.channels + c) * a.dstate;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const float2 v = unpack2(h[j / 2]);
            if (n0 + j < a.dstate) dst[n0 + j] = j % 2 ? v.y : v.x;
        }
    } else {
        float* dst = l.work + item * a.dstate * a.channels + c;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const float2 v = unpack2(h[j / 2]);
            if (n0 + j < a.dstate) dst[static_cast<long long>(n0 + j) * a.channels] = j % 2 ? v.y : v.x;
        }
        if (wn == 0) l.work[l.map.items() * a.dstate * a.channels + item * a.channels + c] = sum_dt;
    }
}

// Over the segments of a sequence, a thread for each (sequence, state column, channel): state <- exp(A sum dt) state + the
// segment's own; each segment's place in `work` takes the state that comes in.
template <bool REVERSE>
__global__ void __launch_bounds__(256)
selective_join_kernel(const SsdScanArgs a, const SeqMap map, float* work, const float* outer) {
    const long long per = static_cast<long long>(a.dstate) * a.channels;
    const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int seq = static_cast<int>(i / per);
    if (seq >= map.rows) return;
    const int n = static_cast<int>((i - seq * per) / a.channels), c = static_cast<int>(i % a.channels);
    long long first, count;
    if (map.cu == nullptr) {
        count = map.per_row();
        first = seq * count;
    } else {
        const long long origin = map.start(seq), len = max(map.start(seq + 1) - origin, 0LL);
        first = origin / map.span + seq;
        count = max((len + map.span - 1) / map.span, 1LL);
    }
    const float* sums = work + map.items() * per;
    const float a2 = a.A[static_cast<long long>(c) * a.dstate + n] * kLog2e;
    float v = outer != nullptr ? outer[(static_cast<long long>(seq) * a.channels + c) * a.dstate + n] : 0.f;
    for (long long k = 0; k < count; ++k) {
        const long long item = first + (REVERSE ? count - 1 - k : k);
        float* at = work + item * per + static_cast<long long>(n) * a.channels + c;
        const float own = *at;
        *at = v;
        v = fmaf(ex2f(a2 * sums[item * a.channels + c]), v, own);
    }
}

// (columns of a warp, warps) for a number of state columns
template <class F>
int with_columns(int dstate, F f) {
    auto is = [&](auto npl, auto nw) { return f(npl, nw); };
    if (dstate <= 8) return is(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
    if (dstate <= 16) return is(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
    if (dstate <= 32) return is(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    if (dstate <= 64) return is(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
    return is(std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{});
}

template <ScanMode kMode>
int launch_walk(const SsdScanArgs& a, ScanLaunch l, bool pairs, cudaStream_t stream) {
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return with_columns(a.dstate, [&](auto npl, auto nw) {
            constexpr int NPL = decltype(npl)::value, NW = decltype(nw)::value;
            // sets of 32 channels in a CTA: several, up to 256 threads, only where that leaves two CTAs per SM
            l.cg = NW >= 8 ? 1 : 8 / NW;
            while (true) {
                l.blocks = scan_blocks(a.channels, a.groups, 32 * l.cg);
                if (l.cg == 1 || l.map.items() * l.blocks.count(a.groups) >= 2LL * sm_count()) break;
                l.cg /= 2;
            }
            const long long ctas = l.map.items() * l.blocks.count(a.groups);
            if (ctas > 0x7fffffffLL) return static_cast<int>(SSD_ERR_RANGE);
            const size_t smem = sizeof(float) * kScanTile * (32 * l.cg * (2 + (kMode == kForward ? NW : 0)) + 2 * NPL * NW);
            auto kernel = pairs ? selective_walk_kernel<T, NPL, NW, true, kMode> : selective_walk_kernel<T, NPL, NW, false, kMode>;
            if (smem > 48 * 1024) {
                static std::atomic<uint64_t> done[2];
                const int rc = set_max_smem_once(reinterpret_cast<const void*>(kernel), 96 * 1024, done[pairs]);
                if (rc != SSD_OK) return rc;
            }
            launch_plain(kernel, static_cast<unsigned>(ctas), 32 * NW * l.cg, smem, stream, a, l);
            return launch_status();
        });
    });
}

}  // namespace

int scan_check(const SsdScanArgs& a) {
    if (a.rows <= 0 || a.tokens < 0 || (a.tokens == 0 && a.cu_seqlens == nullptr) || a.channels <= 0 || a.dstate <= 0 ||
        a.groups <= 0 || a.channels % a.groups != 0)
        return SSD_ERR_SHAPE;
    if (a.dstate > kScanMaxState || a.dtype < SSD_F32 || a.dtype > SSD_F16) return SSD_ERR_UNSUPPORTED;
    if (a.tokens > 0x7fffffff - (1 << 20) || a.rows > 0x7ffffff0) return SSD_ERR_RANGE;
    if (!a.A || (a.tokens > 0 && (!a.x || !a.dt || !a.bm || !a.cm))) return SSD_ERR_NULL;
    return SSD_OK;
}

// A pass over all tokens costs each exponential again.  So sequences are cut only where their channels leave most SMs without
// work, and then into as many segments as fill them.
ScanSegments scan_segments(const SsdScanArgs& a, int per_cta, int slots) {
    const ScanBlocks b = scan_blocks(a.channels, a.groups, per_cta);
    const long long ctas = static_cast<long long>(a.rows) * b.count(a.groups);
    const long long total = a.cu_seqlens ? a.tokens : a.tokens * a.rows;
    ScanSegments s{1 << 30, 0, false};
    if (ctas * 2 < slots && total > 2 * kScanCheckpoint) {
        const long long span = total * b.count(a.groups) / (2LL * slots);
        s.span = static_cast<int>(span < kScanCheckpoint ? kScanCheckpoint
                                                         : (span + kScanCheckpoint - 1) / kScanCheckpoint * kScanCheckpoint);
        s.split = s.span < a.tokens;
    }
    if (!s.split) s.span = 1 << 30;
    s.items = scan_map(a, s.span).items();
    return s;
}

int scan_segment_states(const SsdScanArgs& a, const ScanSegments& s, float* work, const void* dout, const float* dfinal,
                        cudaStream_t stream) {
    ScanLaunch l{scan_map(a, s.span), {}, 1, true, work, dout};
    const bool pairs = [&] {
        const size_t element = a.dtype == SSD_F32 ? 4 : 2;
        return scan_pairs(a, element) && aligned_to(2 * element, dout);
    }();
    const int rc = dout != nullptr ? launch_walk<kStartGradient>(a, l, pairs, stream) : launch_walk<kEndState>(a, l, pairs, stream);
    if (rc != SSD_OK) return rc;
    const long long threads = static_cast<long long>(a.rows) * a.dstate * a.channels, grid = (threads + 255) / 256;
    if (grid > 0x7fffffffLL) return SSD_ERR_RANGE;
    if (dout != nullptr)
        launch_plain(selective_join_kernel<true>, static_cast<unsigned>(grid), 256, 0, stream, a, l.map, work, dfinal);
    else
        launch_plain(selective_join_kernel<false>, static_cast<unsigned>(grid), 256, 0, stream, a, l.map, work, a.initial_state);
    return launch_status();
}

}  // namespace ssd

extern "C" size_t ssd_selective_scan_work_bytes(const SsdScanArgs* args) {
    using namespace ssd;
    if (args == nullptr || scan_check(*args) != SSD_OK) return 0;
    return sizeof(float) * scan_segment_floats(*args, scan_segments(*args, 32, sm_count()));
}

extern "C" size_t ssd_selective_scan_checkpoint_bytes(const SsdScanArgs* args) {
    using namespace ssd;
    if (args == nullptr || scan_check(*args) != SSD_OK) return 0;
    return sizeof(float) * static_cast<size_t>(scan_map(*args, kScanCheckpoint).items()) * args->dstate * args->channels;
}

extern "C" int ssd_selective_scan_fwd(const SsdScanArgs* args, ssd_stream_t stream) {
    using namespace ssd;
    if (args == nullptr) return SSD_ERR_NULL;
    const SsdScanArgs& a = *args;
    if (const int rc = scan_check(a); rc != SSD_OK) return rc;
    if (!a.out && a.tokens > 0) return SSD_ERR_NULL;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const ScanSegments s = scan_segments(a, 32, sm_count());
    if (s.split) {
        if (!a.work) return SSD_ERR_NULL;
        if (const int rc = scan_segment_states(a, s, a.work, nullptr, nullptr, st); rc != SSD_OK) return rc;
    }
    const ScanLaunch l{scan_map(a, s.span), {}, 1, s.split, a.work, nullptr};
    return launch_walk<kForward>(a, l, scan_pairs(a, a.dtype == SSD_F32 ? 4 : 2), st);
}
