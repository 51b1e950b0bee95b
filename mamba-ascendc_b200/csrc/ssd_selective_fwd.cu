// Selective scan, forward, and the segment states that both directions take:
//
//   a_t[n] = exp(dt_t A[n]) ;  h_t[n] = a_t[n] h_{t-1}[n] + dt_t x_t B_t[n] ;  y_t = sum_n C_t[n] h_t[n]   for every channel
//
// What bounds it: instructions.  Each (token, channel, state column) takes an exponential (an SM forms 16 a cycle, eight cycles
// for a warp's), two products and two multiply-adds, each (token, channel) about 45 more for softplus, gate, loads and stores,
// while with 16 columns the bytes are 8 for 16 exponentials.  The walk over the tokens is serial with the state in registers,
// so that each exponential is formed once.
//
// Layout: a lane owns a channel, a warp NPL state columns of 32 channels, the NW warps of a CTA all columns of them.  B and C
// are the same for all lanes (one broadcast load for two tokens of a column), and nothing is exchanged between lanes; the NW
// partial sums of y meet in shared memory.  Tokens pass through shared memory kScanTile at a time: dt (softplus taken once)
// and dt x of two tokens side by side, B and C in fp32.  In long sequences as many warps again stage the next tile and finish the
// last one (gate, skip connection, stores) under the walk: [1,8192,4096] with 16 columns takes 297 us where the same warps
// doing both in turn take 364.  There the exponentials take 0.68 of their rate, shared memory about 0.7; the walk alone takes 228.
//
// kMode: the forward pass itself; each segment's end state from a zero start; or backward in time, the gradient that a segment
// hands to the state before it, e <- a_t (e + C_t dy_t), with dy = dout silu(z).
#include <algorithm>
#include <type_traits>

#include "ssd_selective.cuh"

namespace ssd {

namespace {

constexpr int kScanTile = 32;
constexpr int kTileRow = kScanTile + 2;  // tokens of a column in shared memory, padded
constexpr int kWalkChannels = 32;
enum ScanMode { kForward, kEndState, kStartGradient };

struct ScanLaunch {
    SeqMap map;
    ScanBlocks blocks;
    bool split;            // start states come from `work`
    float* work;           // [items][dstate][channels], [items][channels]
    const void* dout;      // kStartGradient
};

template <int NPL, int NW, ScanMode kMode>
struct WalkTile {
    static constexpr int kCols = NPL * NW;  // state columns, those behind dstate are zeros
    float4 du[kScanTile / 2][kWalkChannels];  // dt of two tokens, dt x (or dy) of them
    float b[kCols][kTileRow];                 // B, or C
    float c[kMode == kForward ? kCols : 1][kTileRow];
    float2 y[kMode == kForward ? NW : 1][kScanTile / 2][kWalkChannels];
};

// What a staging thread loads of a tile.
template <class T, int NPL, int NW>
struct StagedRaw {
    static constexpr int kPairs = 16 / NW, kQuads = NPL / 2;  // pairs of channels, quads of state columns
    Pack<T, 2> x[kPairs], dt[kPairs], z[kPairs];
    Pack<T, 4> q[kQuads];
};

// Where the helpers' loads land: each thread copies what it will read itself, so that its own wait is all there is to wait for.
constexpr int kRing = 3, kHelpTokens = 256;
template <class T, int NPL, int NW>
struct WalkRing {
    using Raw = StagedRaw<T, NPL, NW>;
    Pack<T, 2> x[Raw::kPairs][32 * NW], dt[Raw::kPairs][32 * NW], z[Raw::kPairs][32 * NW];
    Pack<T, 4> q[Raw::kQuads][32 * NW];
};

template <class T, int NPL, int NW, bool HELPED, bool VECTOR, ScanMode kMode>
__global__ void __launch_bounds__(32 * NW * (HELPED ? 2 : 1), HELPED && NPL <= 4 && NW <= 4 && kMode != kForward ? 2 : 1)
selective_walk_kernel(const SsdScanArgs a, const ScanLaunch l) {
    using Tile = WalkTile<NPL, NW, kMode>;
    constexpr int kCols = Tile::kCols, kThreads = 32 * NW;
    constexpr bool kReverse = kMode == kStartGradient;
    extern __shared__ __align__(16) unsigned char walk_smem[];
    Tile* const sms = reinterpret_cast<Tile*>(walk_smem);
    const int blocks = l.blocks.count(a.groups);
    const long long item = blockIdx.x / blocks;
    const ChannelBlock cb = channel_block(l.blocks, blockIdx.x % blocks, a.channels, a.groups);
    Span s;
    if (!locate(l.map, item, s)) return;
    const bool walks = !HELPED || threadIdx.x < kThreads, stages = !HELPED || !walks;
    const int tid = HELPED ? threadIdx.x % kThreads : threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long first_token = (l.map.cu == nullptr ? s.seq * l.map.tokens : 0) + s.origin;

    if (s.pad) {
        if (kMode == kForward)
            for (long long i = threadIdx.x; i < static_cast<long long>(s.t1 - s.t0) * cb.n; i += blockDim.x)
                static_cast<T*>(a.out)[(s.origin + s.t0 + i / cb.n) * a.channels + cb.first + i % cb.n] = from_f<T>(0.f);
        return;
    }

    // ---- the walk's own state
    const int c = cb.first + lane, n0 = warp * NPL;
    const bool live = lane < cb.n;
    float h[NPL], a2[NPL];
    float sum_dt = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int n = n0 + j;
        const bool in = walks && live && n < a.dstate;
        a2[j] = in ? decay_rate(a.A[static_cast<long long>(c) * a.dstate + n]) : 0.f;
        h[j] = 0.f;
        if (kMode == kForward && in) {
            if (l.split)
                h[j] = l.work[(item * a.dstate + n) * a.channels + c];
            else if (a.initial_state != nullptr)
                h[j] = a.initial_state[(static_cast<long long>(s.seq) * a.channels + c) * a.dstate + n];
        }
    }
    const long long checkpoint0 = l.map.cu == nullptr
                                      ? s.seq * ((l.map.tokens + kScanCheckpoint - 1) / kScanCheckpoint)
                                      : s.origin / kScanCheckpoint + s.seq;

    // ---- staging: a thread has two neighbouring channels of kPairs tokens, two neighbouring ones at a time, and quads of
    // state columns of B and C
    using Raw = StagedRaw<T, NPL, NW>;
    constexpr int kPairs = Raw::kPairs, kQuads = Raw::kQuads, kArrayQuads = kScanTile * kCols / 4;
    const int pair = tid & 15, pn = max(min(cb.n - 2 * pair, 2), 0), c2 = cb.first + 2 * pair;
    const auto row_at = [&](int p) { return 2 * ((tid >> 4) + p / 2 * 2 * NW) + p % 2; };
    float2 bias = make_float2(0.f, 0.f), skip = bias;
    if (a.dt_bias != nullptr) bias = make_float2(pn > 0 ? a.dt_bias[c2] : 0.f, pn > 1 ? a.dt_bias[c2 + 1] : 0.f);
    if (a.D != nullptr) skip = make_float2(pn > 0 ? a.D[c2] : 0.f, pn > 1 ? a.D[c2 + 1] : 0.f);
    const Rows<T> xs = kReverse ? Rows<T>(static_cast<const T*>(l.dout) + first_token * a.channels + c2, a.channels)
                                : Rows<T>(static_cast<const T*>(a.x) + first_row(l.map, s, a.x_strides) + c2, a.x_strides[1]);
    const Rows<T> dts(static_cast<const T*>(a.dt) + first_row(l.map, s, a.dt_strides) + c2, a.dt_strides[1]);
    const Rows<T> zs(static_cast<const T*>(a.z) + first_row(l.map, s, a.z_strides) + c2, a.z_strides[1]);
    const Rows<T> bs(static_cast<const T*>(a.bm) + first_row(l.map, s, a.b_strides) + cb.group * a.b_strides[2], a.b_strides[1]);
    const Rows<T> cs(static_cast<const T*>(a.cm) + first_row(l.map, s, a.c_strides) + cb.group * a.c_strides[2], a.c_strides[1]);
    T* out = static_cast<T*>(a.out) + first_token * a.channels + c2;

    Raw raw;
    // quad i of this thread: of B in the first half of their numbers, of C in the second (backwards C takes B's place)
    const auto quad_of_c = [&](int i) { return kReverse || tid + i * kThreads >= kArrayQuads; };
    const auto has_quad = [&](int i) { return kMode == kForward || tid + i * kThreads < kArrayQuads; };
    const auto quad_row = [&](int i) { return (tid + i * kThreads) % kArrayQuads / (kCols / 4); };
    const auto quad_col = [&](int i) { return (tid + i * kThreads) % (kCols / 4) * 4; };
    const auto request = [&](int t0) {
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
            const int t = t0 + row_at(p), n = t < s.t1 ? pn : 0;
            load_raw<VECTOR, false>(raw.x[p], xs.at(t), n);
            load_raw<VECTOR, false>(raw.dt[p], dts.at(t), n);
            if (kReverse && a.z != nullptr) load_raw<VECTOR, false>(raw.z[p], zs.at(t), n);
        }
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
            if (has_quad(i)) {
                const int t = t0 + quad_row(i), n = quad_col(i);
                load_raw<VECTOR, false>(raw.q[i], (quad_of_c(i) ? cs : bs).at(t) + n, t < s.t1 ? min(a.dstate - n, 4) : 0);
            }
    };
    const int tiles = (s.t1 - s.t0 + kScanTile - 1) / kScanTile;
    const auto tile_start = [&](int k) { return s.t0 + (kReverse ? tiles - 1 - k : k) * kScanTile; };
    float2 held[kPairs];  // x, for the skip connection
    const auto stage = [&](Tile& sm, int t0) {
        const int nt = s.t1 - t0;
#pragma unroll
        for (int p = 0; p < kPairs; p += 2) {
            float2 d[2], u[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 xv = pair_f(raw.x[p + i]);
                d[i] = pair_f(raw.dt[p + i]);
                d[i] = make_float2(d[i].x + bias.x, d[i].y + bias.y);
                if (a.softplus) d[i] = make_float2(softplus_series(d[i].x), softplus_series(d[i].y));
                if (row_at(p + i) >= nt) d[i] = make_float2(0.f, 0.f);  // behind the last token the state stays
                if (kReverse) {
                    u[i] = xv;
                    if (a.z != nullptr) {
                        const float2 zv = pair_f(raw.z[p + i]);
                        u[i] = make_float2(xv.x * zv.x * sigmoid_fast(zv.x), xv.y * zv.y * sigmoid_fast(zv.y));
                    }
                } else {
                    u[i] = make_float2(d[i].x * xv.x, d[i].y * xv.y);
                }
                held[p + i] = xv;
            }
            float4* at = &sm.du[row_at(p) / 2][2 * pair];
            at[0] = make_float4(d[0].x, d[1].x, u[0].x, u[1].x);
            at[1] = make_float4(d[0].y, d[1].y, u[0].y, u[1].y);
        }
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
            if (has_quad(i)) {
                float* dst = (kMode == kForward && quad_of_c(i) ? sm.c : sm.b)[quad_col(i)] + quad_row(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) dst[j * kTileRow] = to_f(raw.q[i].v[j]);
            }
    };
    // what the outputs of a tile take beside the sums
    const auto request_gate = [&](int t0) {
        if (kMode != kForward || a.z == nullptr) return;
#pragma unroll
        for (int p = 0; p < kPairs; ++p) load_raw<VECTOR, false>(raw.z[p], zs.at(t0 + row_at(p)), t0 + row_at(p) < s.t1 ? pn : 0);
    };
    const auto finish = [&](const Tile& sm, int t0) {
        const int nt = s.t1 - t0;
        T* to = out + static_cast<long long>(t0) * a.channels;
#pragma unroll
        for (int p = 0; p < kPairs; p += 2) {
            const int row = row_at(p);
            float4 y = make_float4(skip.x * held[p].x, skip.x * held[p + 1].x, skip.y * held[p].y, skip.y * held[p + 1].y);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(&sm.y[kMode == kForward ? w : 0][row / 2][2 * pair]);
                y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
            }
            float2 o[2] = {make_float2(y.x, y.z), make_float2(y.y, y.w)};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (a.z != nullptr) {
                    const float2 zv = pair_f(raw.z[p + i]);
                    o[i].x *= zv.x * sigmoid_fast(zv.x);
                    o[i].y *= zv.y * sigmoid_fast(zv.y);
                }
                store_pair<VECTOR>(to + static_cast<long long>(row + i) * a.channels, o[i], row + i < nt ? pn : 0);
            }
        }
    };
    const auto walk_tile = [&](Tile& sm, int t0) {
        const int nt = min(s.t1 - t0, kScanTile);
        if (kMode == kForward && a.checkpoints != nullptr && (t0 - s.t0) % kScanCheckpoint == 0 && live) {
            float* dst = a.checkpoints + (checkpoint0 + t0 / kScanCheckpoint) * a.dstate * a.channels + c;
#pragma unroll
            for (int j = 0; j < NPL; ++j)
                if (n0 + j < a.dstate) dst[static_cast<long long>(n0 + j) * a.channels] = h[j];
        }
        // kGroup tokens at a time.  Only the states depend on the token before: the operands of the next groups are on their
        // way, and the next one's exponentials lie between the steps of this one's recurrence, all in one straight line.
        // Groups of four or eight tokens take 1% longer with helpers and up to 10% without.  Rows behind the last token have
        // dt = 0; where they are half of the tile they are left out.
        constexpr int kGroup = 2, kAhead = NPL <= (HELPED ? 4 : 2) ? 2 : 1;
        struct Operands {
            float dt[kGroup], u[kGroup], b[NPL][kGroup], c[NPL][kGroup];
        };
        const auto walk = [&](auto rows) {
            constexpr int kRows = decltype(rows)::value, kGroups = kRows / kGroup;
            const auto fetch = [&](Operands& o, int group) {
                const int first = (kReverse ? kGroups - 1 - group : group) * kGroup;
#pragma unroll
                for (int i = 0; i < kGroup; i += 2) {
                    const float4 du = sm.du[(first + i) / 2][lane];
                    o.dt[i] = du.x, o.dt[i + 1] = du.y, o.u[i] = du.z, o.u[i + 1] = du.w;
                }
#pragma unroll
                for (int j = 0; j < NPL; ++j) {
                    const float2 bv = *reinterpret_cast<const float2*>(&sm.b[n0 + j][first]);
                    o.b[j][0] = bv.x, o.b[j][1] = bv.y;
                    if (kMode == kForward) {
                        const float2 cv = *reinterpret_cast<const float2*>(&sm.c[kMode == kForward ? n0 + j : 0][first]);
                        o.c[j][0] = cv.x, o.c[j][1] = cv.y;
                    }
                }
            };
            Operands now, next, third;
            float e[NPL][kGroup], e_next[NPL][kGroup];
            fetch(now, 0);
            if (kAhead == 2 && kGroups > 1) fetch(next, 1);
#pragma unroll
            for (int j = 0; j < NPL; ++j)
#pragma unroll
                for (int i = 0; i < kGroup; ++i) e[j][i] = decay(now.dt[i], a2[j]);
#pragma unroll
            for (int group = 0; group < kGroups; ++group) {
                if (group + kAhead < kGroups) fetch(kAhead == 2 ? third : next, group + kAhead);
                float in[NPL][kGroup], y[kGroup];
#pragma unroll
                for (int j = 0; j < NPL; ++j)
#pragma unroll
                    for (int i = 0; i < kGroup; ++i) {
                        in[j][i] = now.u[i] * now.b[j][i];
                        if (kReverse) in[j][i] *= e[j][i];
                    }
#pragma unroll
                for (int i = 0; i < kGroup; ++i) {
                    const int t = kReverse ? kGroup - 1 - i : i;
                    if (kMode != kForward) sum_dt += now.dt[t];
#pragma unroll
                    for (int j = 0; j < NPL; ++j) {
                        h[j] = fmaf(e[j][t], h[j], in[j][t]);
                        if (kMode == kForward) y[t] = j == 0 ? now.c[0][t] * h[0] : fmaf(now.c[j][t], h[j], y[t]);
                    }
                    if (group + 1 < kGroups) {
#pragma unroll
                        for (int j = 0; j < NPL; ++j) e_next[j][t] = decay(next.dt[t], a2[j]);
                    }
                }
                if (kMode == kForward) {
#pragma unroll
                    for (int i = 0; i < kGroup; i += 2)
                        sm.y[kMode == kForward ? warp : 0][(group * kGroup + i) / 2][lane] = make_float2(y[i], y[i + 1]);
                }
#pragma unroll
                for (int j = 0; j < NPL; ++j)
#pragma unroll
                    for (int i = 0; i < kGroup; ++i) e[j][i] = e_next[j][i];
                now = next;
                if (kAhead == 2) next = third;
            }
        };
        if (nt > kScanTile / 2)
            walk(std::integral_constant<int, kScanTile>{});
        else
            walk(std::integral_constant<int, kScanTile / 2>{});
    };

    if constexpr (HELPED) {
        // The helpers are a tile ahead of the walk with its operands and one behind it with the outputs; what they load is on
        // its way for two tiles.  (Registers in place of the ring: 340 us against 302, as later loads hold up earlier ones.)
        auto* const ring = reinterpret_cast<WalkRing<T, NPL, NW>*>(sms + 2);
        const auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(2 * kThreads) : "memory"); };
        if (walks) {
            meet();
            for (int k = 0; k < tiles; ++k) {
                walk_tile(sms[k & 1], tile_start(k));
                meet();
            }
        } else {
            const auto copy = [&](int k) {  // of a tile, an empty group behind the last one
                if (k < tiles) {
                    auto& to = ring[k % kRing];
                    const int t0 = tile_start(k);
#pragma unroll
                    for (int p = 0; p < kPairs; ++p) {
                        const int t = min(t0 + row_at(p), s.t1 - 1);
                        const bool in = t0 + row_at(p) < s.t1 && pn > 0;
                        copy_async(to.x[p][tid], xs.at(t), in);
                        copy_async(to.dt[p][tid], dts.at(t), in);
                        if (kMode != kEndState && a.z != nullptr) copy_async(to.z[p][tid], zs.at(t), in);
                    }
#pragma unroll
                    for (int i = 0; i < kQuads; ++i)
                        if (has_quad(i)) {
                            const int t = min(t0 + quad_row(i), s.t1 - 1), n = quad_col(i);
                            copy_async(to.q[i][tid], (quad_of_c(i) ? cs : bs).at(t) + n, t0 + quad_row(i) < s.t1 && n < a.dstate);
                        }
                }
                copies_commit();
            };
            const auto prepare = [&](int k) {
                copies_wait<kRing - 2>();
                const auto& from = ring[k % kRing];
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    raw.x[p] = from.x[p][tid], raw.dt[p] = from.dt[p][tid];
                    if (kReverse && a.z != nullptr) raw.z[p] = from.z[p][tid];
                }
#pragma unroll
                for (int i = 0; i < kQuads; ++i)
                    if (has_quad(i)) raw.q[i] = from.q[i][tid];
                stage(sms[k & 1], tile_start(k));
            };
            const auto conclude = [&](int k) {
                if (kMode != kForward) return;
                const auto& from = ring[k % kRing];
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    held[p] = pair_f(from.x[p][tid]);
                    if (a.z != nullptr) raw.z[p] = from.z[p][tid];
                }
                finish(sms[k & 1], tile_start(k));
            };
            for (int k = 0; k < kRing - 1; ++k) copy(k);
            if (tiles > 0) prepare(0);
            meet();
            for (int k = 0; k < tiles; ++k) {
                if (k > 0) conclude(k - 1);
                copy(k + kRing - 1);
                if (k + 1 < tiles) prepare(k + 1);
                meet();
            }
            if (tiles > 0) conclude(tiles - 1);
            return;
        }
    } else {
        if (tiles > 0) request(tile_start(0));
        for (int k = 0; k < tiles; ++k) {
            stage(sms[0], tile_start(k));
            __syncthreads();
            if (k + 1 < tiles) request(tile_start(k + 1));
            request_gate(tile_start(k));
            walk_tile(sms[0], tile_start(k));
            __syncthreads();
            if (kMode == kForward) finish(sms[0], tile_start(k));
        }
    }
    if (!live) return;
    if (kMode == kForward) {
        if (!s.last || a.final_state == nullptr) return;
        float* dst = a.final_state + (static_cast<long long>(s.seq) * a.channels + c) * a.dstate;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (n0 + j < a.dstate) dst[n0 + j] = h[j];
    } else {
        float* dst = l.work + item * a.dstate * a.channels + c;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (n0 + j < a.dstate) dst[static_cast<long long>(n0 + j) * a.channels] = h[j];
        if (warp == 0) l.work[l.map.items() * a.dstate * a.channels + item * a.channels + c] = sum_dt;
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
    const float a2 = decay_rate(a.A[static_cast<long long>(c) * a.dstate + n]);
    float v = outer != nullptr ? outer[(static_cast<long long>(seq) * a.channels + c) * a.dstate + n] : 0.f;
    for (long long k = 0; k < count; ++k) {
        const long long item = first + (REVERSE ? count - 1 - k : k);
        float* at = work + item * per + static_cast<long long>(n) * a.channels + c;
        const float own = *at;
        *at = v;
        v = fmaf(decay(sums[item * a.channels + c], a2), v, own);
    }
}

// (columns of a warp, warps, helped) for a number of state columns.  Without helpers (odd alignments, sequences of a few tiles) and
// with `few` CTAs, no more than SMs, four columns per warp leave a scheduler with one warp that also has to stage: two
// columns per warp then, although each warp reads dt and dt x again (368 against 420 us for [1,8192,4096] with 16 columns).
// With helpers, against without (us):   16 columns  [1,8192,4096] 297 / 364   [4,2000,2048] 129 / 142   [1,16384,1536] 316 / 402
//   8 columns [1,8192,4096] 241 / 325   32 columns [1,8192,4096] 471 / 536   64 columns [1,4096,4096] 417 / 478.
// With 128 columns there are none: in fp32 the two tiles and the ring would take 287 KB, and in 16 bits, where they take 219, sixteen
// warps leave a thread 128 registers, in which the forward walk spills 164 bytes (255 registers without staging warps).
template <class F>
int with_columns(int dstate, bool few, bool help, F f) {
    const auto is = [&](auto npl, auto nw) { return help ? f(npl, nw, std::true_type{}) : f(npl, nw, std::false_type{}); };
    if (dstate <= 8 && few) return is(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
    if (dstate <= 8) return is(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
    if (dstate <= 16 && few && !help) return f(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{}, std::false_type{});
    if (dstate <= 16) return is(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
    if (dstate <= 32) return is(std::integral_constant<int, 4>{}, std::integral_constant<int, 8>{});
    if (dstate <= 64) return is(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{}, std::false_type{});
}

template <ScanMode kMode>
int launch_walk(const SsdScanArgs& a, ScanLaunch l, bool pairs, cudaStream_t stream) {
    l.blocks = scan_blocks(a.channels, a.groups, kWalkChannels);
    const long long ctas = l.map.items() * l.blocks.count(a.groups);
    if (ctas > 0x7fffffffLL) return SSD_ERR_RANGE;
    // Helpers pay where there are tiles enough to be ahead: with and without, [64,64,2048] takes 86 and 73 us, [8,128,2048] and
    // [8,256,2048] 24 and 40 both ways, [8,512,2048] 70.6 and 74.8.
    const long long mean = l.map.cu == nullptr ? a.tokens : a.tokens / a.rows;
    const bool help = pairs && std::min<long long>(mean, l.map.span) >= kHelpTokens;
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return with_columns(a.dstate, ctas <= sm_count(), help, [&](auto npl, auto nw, auto helped) {
            constexpr bool kHelped = decltype(helped)::value;
            constexpr int NPL = decltype(npl)::value, NW = decltype(nw)::value;
            constexpr size_t smem = kHelped ? 2 * sizeof(WalkTile<NPL, NW, kMode>) + kRing * sizeof(WalkRing<T, NPL, NW>)
                                            : sizeof(WalkTile<NPL, NW, kMode>);
            const auto kernel = pairs ? selective_walk_kernel<T, NPL, NW, kHelped, true, kMode>
                                      : selective_walk_kernel<T, NPL, NW, false, false, kMode>;
            if (smem > 48 * 1024) {
                static std::atomic<uint64_t> done[2];
                const int rc = set_max_smem_once(reinterpret_cast<const void*>(kernel), smem, done[pairs]);
                if (rc != SSD_OK) return rc;
            }
            launch_plain(kernel, static_cast<unsigned>(ctas), 32 * NW * (kHelped ? 2 : 1), smem, stream, a, l);
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
    if (!row_steps(a.x_strides[1], a.dt_strides[1], a.z_strides[1], a.b_strides[1], a.c_strides[1], a.channels,
                   static_cast<int64_t>(a.groups) * a.dstate))
        return SSD_ERR_RANGE;
    if (!a.A || (a.tokens > 0 && (!a.x || !a.dt || !a.bm || !a.cm))) return SSD_ERR_NULL;
    return SSD_OK;
}

// A pass over all tokens costs each exponential again.  So sequences are cut only where their channels leave most SMs without
// work, and then into as many segments as fill them.
ScanSegments scan_segments(const SsdScanArgs& a, int per_cta, int slots) {
    const ScanBlocks b = scan_blocks(a.channels, a.groups, per_cta);
    const long long ctas = static_cast<long long>(a.rows) * b.count(a.groups);
    const long long total = a.cu_seqlens ? a.tokens : a.tokens * a.rows;
    constexpr int kWhole = 0x7fffffff;  // more than any sequence has
    ScanSegments s{kWhole, 0, false};
    if (ctas * 2 < slots && total > 2 * kScanCheckpoint) {
        const long long span = total * b.count(a.groups) / (2LL * slots);
        s.span = static_cast<int>(span < kScanCheckpoint ? kScanCheckpoint
                                                         : (span + kScanCheckpoint - 1) / kScanCheckpoint * kScanCheckpoint);
        s.split = s.span < a.tokens;
    }
    if (!s.split) s.span = kWhole;
    s.items = scan_map(a, s.span).items();
    return s;
}

int scan_segment_states(const SsdScanArgs& a, const ScanSegments& s, float* work, const void* dout, const float* dfinal,
                        cudaStream_t stream) {
    ScanLaunch l{scan_map(a, s.span), {}, true, work, dout};
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
    const ScanLaunch l{scan_map(a, s.span), {}, s.split, a.work, nullptr};
    return launch_walk<kForward>(a, l, scan_pairs(a, a.dtype == SSD_F32 ? 4 : 2), st);
}
