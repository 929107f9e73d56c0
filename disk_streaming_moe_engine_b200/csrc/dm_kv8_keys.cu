// dm_kv8_keys.cu — attention over the 8-bit paged cache with the keys on the tensor cores' M
// side: one token (or a few query rows) per request against long caches, any type.
//
// Work: an item is RB query rows (a row = one query token and one query head) of one request
// and kv head; its keys come in tiles of 128 tokens (8 pages).  Per tile, on tcgen05 with
// e4m3 operands straight from the cache's bytes (no conversion of the cache at all):
//   S^T [128 tokens x N] = codeK [128 x D] . Qterms^T [D x N]
//   O^T [D x NP]        += codeV^T [D x 128] . Pterms [128 x NP]
// N = RB rows x TERMS columns: q and the softmax weights enter as sums of e4m3 terms, term i
// scaled by 2^-4i in columns of its own, so a term adds 4 bits (at least 2^-4 of what the terms
// before it left) and costs only N: 2 terms hold bf16's 8 bits of q, its weights take 3 (2^-10, so
// that the result is as good as its rounding; 2 were 2 to 4 % faster), fp32 5 for both (2^-20).
// Weights need range as well: thousands of keys may lie many nats below one whose V is small.  So NP
// is twice their terms: a weight below 2^-12 of the reference enters 2^14 times larger in columns of
// its own, the others' columns hold zero there (one group of columns lost all below 2^-19).  The tensor
// time of a tile is that of reading 128 x 32 operand bytes per instruction whatever N <= 64 is, far
// below the time of the tile's bytes from HBM, which is what bounds long caches: 64 requests of
// 32768 tokens (2 kv heads of 256, 8 query heads each) take 348 us in a graph, 6.2 TB/s or 0.96 of the
// measured copy bandwidth, 367 us called with cold inputs.  Short ones are bound by the chain of waits
// of one tile (0.65 us and more) and of an item's start, end and join (2 to 4 us): one request of 4096
// tokens takes 19 us.
//
// Softmax in base 2: with a page's scales sK, sV = 2^v,
//   x = q . k (scaled, in log2 units),  w = 2^(x + v - M),  o = sum w codeV / sum w 2^-v,
// M the row's reference for x + v: raised to the running maximum whenever some x + v exceeds
// it by more than 2 (then O^T and the sums are rescaled).  Scores and references are kept in halves of
// log2 units: e = 2^((x + v - M) / 2) does not underflow where w = e e does, and a key whose w is far
// below 2^-126 may well have its share (e 2^-v) e of the sum, as pages of zeros do (their scale is
// 2^-100).  So w <= 4 and 64 w stays in e4m3's
// range whatever the scales are; three terms leave an error of at most 2^-10 w down to w = 2^-26,
// below that 2^-37 (five: 2^-20 w, 2^-46).  Thread t of
// a group of 128 owns token t of the tile for 8 of the rows: scores, weights, its share of the row
// sums; only the reference crosses threads.
//
// Split: all items' tiles in one sequence, cut into one contiguous range per CTA (one or two per
// SM, persistent), so ragged lengths balance to a tile.  An item cut by a range boundary
// leaves partial O, M, sum in the workspace, and the last of its CTAs to arrive joins them in
// range order: the result does not depend on timing.
//
// Roles: RB / 8 groups of 4 warps for softmax, epilogue and Q preparation; a producer warp
// (groups of 4 tiles, a lane per page: page ids and scales fetched groups ahead, one TMA box per
// page; a missing page reads zeros); an MMA warp (one thread).  All waits are bounded; after a
// timeout every role leaves and copies and MMAs in flight are waited for.
#include <atomic>
#include <cmath>

#include "dm_kv8_walk.cuh"

namespace dm {

constexpr int kKeySmem = 227 * 1024;         // shared memory of an SM for its CTAs
constexpr int kKeyLead = 1;                  // an item's start and end in tiles (KeyWalk)
constexpr float kKeyLazy = 1.0f;             // what a weight may exceed the reference by, in halves of log2 units
constexpr float kKeyBoost = 64.0f;           // weights enter as 64 w <= 256
constexpr float kKeySmall = 1.0f / 64;       // e of those in the second group of columns, below 2^-12 and
constexpr float kKeyGroup = 16384.0f;        // times 2^14

template <typename T, int D, int RB, int CTAS>
struct KeyShape {
    static constexpr int kTerms = sizeof(T) == 4 ? 5 : 2;    // of q
    static constexpr int kPTerms = sizeof(T) == 4 ? 5 : 3;   // of the weights
    static constexpr int kN = (RB * kTerms + 15) / 16 * 16;  // columns behind the terms are never read
    static constexpr int kSoft = RB * 16;                    // softmax threads
    static constexpr int kThreads = kSoft + 64;
    static constexpr int CW = D >= 128 ? 128 : D;
    static constexpr int kChunks = D / CW;
    static constexpr int kNP = 2 * RB * kPTerms;             // per term and 8 rows: 8 columns of each group
    static constexpr int kQ = kN * D;
    static constexpr int kP = kNP * kKeyTile;                // one buffer
    static constexpr int kCtas = CTAS;                       // per SM
    using Tile = KeyTile<D, true>;                    // K and V of a tile
    static constexpr int kSlot = Tile::kSlot;
    static constexpr int fixed(int bufs) { return kQ + bufs * kP + 1024; }
    static constexpr int slots(int bufs) {
        const int fit = (kKeySmem / kCtas - 6144 - fixed(bufs)) / kSlot;  // static arrays and 1 KB per CTA beside it
        return fit > kKeyMaxSlots ? kKeyMaxSlots : fit;
    }
    // Buffers of the scores and of the weights: two, so that no role waits, unless the second costs
    // a slot of the ring (fp32 at D = 256: 32 requests of 8000 keys 82 us with two buffers and two
    // slots, 67 with one and three) or does not fit tensor memory.
    static constexpr int kBufs = slots(2) == slots(1) && (2 * kN + kChunks * kNP) * CTAS <= 512 ? 2 : 1;
    static constexpr int kSlots = slots(kBufs);
    static constexpr size_t kSmem = static_cast<size_t>(kSlots) * kSlot + fixed(kBufs);
    static constexpr int kColsUsed = kBufs * kN + kChunks * kNP;
    static constexpr int kCols = kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
    static_assert(kSlots >= 2 && kN % 16 == 0 && kNP % 16 == 0 && kColsUsed * kCtas <= 512, "shape");
    static_assert(kQ % 1024 == 0 && kP % 1024 == 0, "tiles start at the swizzle's 1024 bytes");
};

struct KeyArgs {
    CUtensorMap map;
    Kv8AttnArgs a;
};

template <typename T, int D, int RB, int CTAS>
__global__ void __launch_bounds__(KeyShape<T, D, RB, CTAS>::kThreads, KeyShape<T, D, RB, CTAS>::kCtas)
    kv8_attn_keys_kernel(const __grid_constant__ KeyArgs ka) {
    using S = KeyShape<T, D, RB, CTAS>;
    constexpr int N = S::kN, NP = S::kNP, TERMS = S::kTerms, PT = S::kPTerms, BUFS = S::kBufs, CW = S::CW, SL = S::kSlots, SOFT = S::kSoft;
    constexpr uint32_t kO = BUFS * N;  // tensor memory columns: scores, O
    constexpr int NT = S::kThreads, W_LOAD = SOFT / 32, W_MMA = W_LOAD + 1;
    const Kv8AttnArgs& a = ka.a;
    extern __shared__ __align__(1024) uint8_t key_smem[];
    uint8_t* sm = key_smem + ((1024u - (smem_u32(key_smem) & 1023u)) & 1023u);
    uint8_t* s_q = sm + SL * S::kSlot;
    uint8_t* s_p = s_q + S::kQ;
    __shared__ __align__(8) KeyRing<SL, true> ring;
    __shared__ __align__(8) uint64_t s_full[BUFS], s_free, p_ready[BUFS], pv_done[BUFS], q_ready, done_bar;
    __shared__ float s_frow[RB];
    __shared__ int s_lim[RB];
    // elements of out and of lse of the item's rows, by the item's parity: some threads still write
    // an item's results when others are at the next item's q
    __shared__ int64_t s_off[2][RB], s_lse[2][RB];
    __shared__ float s_red[4][RB], s_fac[32][RB];
    __shared__ long long s_sum[64];
    __shared__ KeyRange s_range;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ int s_nan;  // a NaN code of V that not every row sees was left out of the item's O
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int* abort_flag = &s_abort;

    if (tid == 0) {
        ring.init();
        for (int i = 0; i < BUFS; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], SOFT);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(&s_free, SOFT);
        mbar_init(&q_ready, SOFT);
        mbar_init(&done_bar, 1);
        mbar_fence_init();
        s_abort = 0;
        s_nan = 0;
    }
    if (warp == W_MMA) tc_alloc(&s_tmem, S::kCols);

    tc_fence_before();
    // one tile and its item cost per CTA at least
    const bool active = key_range<RB, kKeyLead, NT>(a, 1 + kKeyLead, s_sum, &s_range);
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    // tile x has buffer x % BUFS, in the phase of this parity
    auto phase = [](uint32_t x) { return x / BUFS & 1u; };

    if (warp == W_LOAD) {
        if (active) key_produce<RB, kKeyLead, D, SL, true>(a, &ka.map, sm, ring, s_range, abort_flag);
        if (a.fill) key_fill<T, D>(a);
    } else if (active && warp == W_MMA) {
        // ---------------- MMA ----------------
        if (lane == 0) {
            uint32_t t = 0, item = 0;
            bool ok = true;
            const uint32_t i_s = f8_idesc(128, N, false, false), i_o = f8_idesc(128, NP, true, true);
            const uint32_t sq = smem_u32(s_q), sp = smem_u32(s_p);
            auto scores = [&](uint32_t x) {  // S^T of tile x into its buffer
                const uint32_t ld = ring.k_load(x);
                ok = ring.wait_full(ld, a.err, abort_flag) &&
                     (BUFS == 2 || x == 0 || mbar_wait_bounded(&s_free, (x - 1) & 1u, a.err, abort_flag));
                if (!ok) return;
                tc_fence_after();
                const uint32_t k = smem_u32(sm + (ld % SL) * S::kSlot);
#pragma unroll
                for (int c = 0; c < S::kChunks; ++c) {
                    const uint64_t ad = f8_desc_k<CW>(k + c * S::Tile::kChunk, S::Tile::kGroup);
                    const uint64_t bd = f8_desc_k<CW>(sq + c * (N * CW), 8 * CW);
#pragma unroll
                    for (int j = 0; j < CW / 32; ++j) f8_mma(tmem + x % BUFS * N, ad + 2 * j, bd + 2 * j, i_s, c > 0 || j > 0);
                }
                tc_commit(&s_full[x % BUFS]);
            };
            KeyWalk<RB, kKeyLead> w(a, s_range);
            while (w.unit < w.end && ok) {
                int first, last, real;
                w.span(first, last, real);
                const int nt = last - first;
                if (nt > 0) {
                    if (!(ok = mbar_wait_bounded(&q_ready, item & 1u, a.err, abort_flag))) break;
                    ++item;
                    tc_fence_after();
                    scores(t);
                    for (int i = 0; i < nt && ok; ++i) {
                        const uint32_t x = t + i;
                        if (i + 1 < nt) scores(x + 1);
                        if (!ok || !(ok = mbar_wait_bounded(&p_ready[x % BUFS], phase(x), a.err, abort_flag))) break;
                        tc_fence_after();
                        const uint32_t ld = ring.v_load(x);
                        const uint32_t v = smem_u32(sm + (ld % SL) * S::kSlot) + S::Tile::kV;
                        const uint64_t bd = f8_desc_n16(sp + x % BUFS * S::kP, kKeyTile * 16);
#pragma unroll
                        for (int c = 0; c < S::kChunks; ++c) {
                            // 64 wide: M rows 64-127 repeat rows 0-63
                            const uint64_t ad = f8_desc_m<CW>(v + c * S::Tile::kChunk, 0, S::Tile::kGroup);
#pragma unroll
                            for (int j = 0; j < kKeyTile / 32; ++j)
                                f8_mma(tmem + kO + c * NP, ad + j * (4 * S::Tile::kGroup / 16), bd + j * (32 * 16 / 16), i_o, i > 0 || j > 0);
                        }
                        tc_commit(&ring.empty[ld % SL]);
                        tc_commit(&pv_done[x % BUFS]);
                    }
                    t += nt;
                }
                w.next();
            }
            tc_commit(&done_bar);
            mbar_wait_bounded(&done_bar, 0, a.err, nullptr);
        }
    } else if (active) {
        // ---------------- softmax, epilogue, Q ----------------
        const int tt = tid & 127, r0 = tid / 128 * 8, wq = warp & 3;  // token, first row, warp of the group
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * wq) << 16) + r0;
        const uint32_t o_lanes = tmem + (static_cast<uint32_t>(32 * wq) << 16) + kO + 2 * r0;
        uint32_t t = 0;
        int item = 0;
        bool ok = true;     // of this thread; all leave together, after a barrier that ORs !ok
        bool left = false;
        KeyWalk<RB, kKeyLead> w(a, s_range);
        while (w.unit < w.end) {
            int lim_min, lim_max;
            key_limits<RB>(a, w.r, w.block(), lim_min, lim_max);
            int t_begin, t_end, real;
            w.span(t_begin, t_end, real);
            const int nt = t_end - t_begin;
            if (nt <= 0) {
                w.next();
                continue;
            }
            const int nrow = min(RB, w.r.m * a.group - w.block() * RB);
            {   // Q terms: 16 threads per row
                constexpr int E = D / 16;
                const int r = tid / 16, e0 = (tid % 16) * E;
                const int f = w.block() * RB + min(r, nrow - 1);
                const int tok = f / a.group, head = w.h * a.group + f % a.group;
                const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(w.r.row0 + tok) * a.q_rs +
                             static_cast<int64_t>(head) * a.q_hs + e0;
                float x[E];
                float amax = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = r < nrow ? static_cast<float>(q[e]) : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (!(fabsf(x[e]) <= 3.402823466e38f)) x[e] = __int_as_float(0x7fc00000);
                    amax = fmaxf(amax, fabsf(x[e]));
                }
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                // largest magnitude of the row to [2^7, 2^8)
                const int ex = max(-120, min(120, (__float_as_int(amax) >> 23) - 127 - 7));
                const float mul = __int_as_float((127 - ex) << 23);
                if (tid % 16 == 0) {
                    s_frow[r] = 0.5f * a.scale_log2 * __int_as_float((127 + ex) << 23);
                    s_lim[r] = r < nrow ? min(w.r.len, max(0, w.r.full - w.r.m + tok + 1)) : 0;
                    s_off[item & 1][r] = static_cast<int64_t>(w.r.row0 + tok) * a.o_rs + static_cast<int64_t>(head) * a.o_hs;
                    s_lse[item & 1][r] = static_cast<int64_t>(w.r.row0 + tok) * a.Hq + head;
                }
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] *= mul;
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    uint32_t lo[TERMS], hi[TERMS];
                    e4m3_split2<TERMS>(x[e], x[e + 1], lo);
                    e4m3_split2<TERMS>(x[e + 2], x[e + 3], hi);
                    const int d = e0 + e;
#pragma unroll
                    for (int i = 0; i < TERMS; ++i)
                        *reinterpret_cast<uint32_t*>(s_q + (d / CW) * (N * CW) + f8_unit<CW>(i * RB + r, (d % CW) / 16) +
                                                     d % 16) = lo[i] | (hi[i] << 16);
                }
                fence_proxy_async_smem();
                mbar_arrive(&q_ready);
                named_bar_sync(1, SOFT);
            }
            float mref[8], l[8], frow[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) mref[r] = -INFINITY, l[r] = 0.0f, frow[r] = s_frow[r0 + r];

            for (int i = 0; i < nt; ++i) {
                const uint32_t x = t + i;
                const int key = (t_begin + i) * kKeyTile + tt;
                // the tile's scales, its scores, and (of two buffers, from the third tile on) the P
                // buffer, tried together since they are mostly there
                const bool t1 = ring.try_meta(x);
                const bool t2 = mbar_try_wait(&s_full[x % BUFS], phase(x));
                const bool t3 = BUFS == 1 || i < 2 || mbar_try_wait(&pv_done[x % BUFS], phase(x - 2));
                if (!(t1 && t2 && t3)) {
                    ok = ok && ring.wait_meta(x, a.err, abort_flag) &&
                         mbar_wait_bounded(&s_full[x % BUFS], phase(x), a.err, abort_flag) &&
                         (BUFS == 1 || i < 2 || mbar_wait_bounded(&pv_done[x % BUFS], phase(x - 2), a.err, abort_flag));
                }
                __syncwarp();  // the loads below are the whole warp's
                tc_fence_after();
                const float2 sc = ring.meta[x % ring.kMeta][tt >> 4];
                const float vexp = static_cast<float>(((__float_as_int(sc.y) >> 23) & 0xff) - 127);
                float y[8];
                {
                    float c[TERMS][8];
#pragma unroll
                    for (int b = 0; b < TERMS; ++b) tc_ld8(lanes + x % BUFS * N + b * RB, c[b]);
                    tc_wait_ld();
                    if constexpr (BUFS == 1) {
                        tc_fence_before();
                        mbar_arrive(&s_free);
                    }
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        y[r] = c[0][r];
#pragma unroll
                        for (int b = 1; b < TERMS; ++b) y[r] = fmaf(c[b][r], 1.0f / static_cast<float>(1 << (4 * b)), y[r]);
                        y[r] = fmaf(y[r], frow[r] * sc.x, 0.5f * vexp);
                    }
                }
                const bool edge = (t_begin + i + 1) * kKeyTile > lim_min;
                bool over = !ok;
                if (edge) {
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (key >= s_lim[r0 + r]) y[r] = -INFINITY;
                }
                if (sc.y < 0.0f) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) y[r] = -INFINITY;
                }
#pragma unroll
                for (int r = 0; r < 8; ++r) over = over || y[r] > mref[r] + kKeyLazy;
                if (named_bar_or(1, SOFT, over)) {
                    // raise the references to the maximum of this tile and rescale; after a failed
                    // wait all threads leave together here
                    if (ok && i > 0)
                        ok = mbar_wait_bounded(&pv_done[(x - 1) % BUFS], phase(x - 1), a.err, abort_flag);
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const float mx = warp_max(y[r]);
                        if (lane == 0) s_red[wq][r0 + r] = mx;
                    }
                    if ((left = named_bar_or(1, SOFT, !ok))) break;
                    float fac[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const float mx = fmaxf(fmaxf(s_red[0][r0 + r], s_red[1][r0 + r]), fmaxf(s_red[2][r0 + r], s_red[3][r0 + r]));
                        const float nm = fmaxf(mref[r], mx);
                        const float f = nm == mref[r] ? 1.0f : exp2f(mref[r] - nm);
                        mref[r] = nm;
                        l[r] = l[r] * f * f;
                        fac[r] = f * f;
                    }
                    if (i > 0) {
                        tc_fence_after();
#pragma unroll 1  // rare: little code
                        for (int c = 0; c < S::kChunks; ++c)
#pragma unroll(PT == 3 ? 2 : 1)
                            for (int b = 0; b < 2 * PT; ++b) {
                                float o[8];
                                const uint32_t at = o_lanes + c * NP + (b >> 1) * (2 * RB) + (b & 1) * 8;
                                tc_ld8(at, o);
                                tc_wait_ld();
#pragma unroll
                                for (int r = 0; r < 8; ++r) o[r] *= fac[r];
                                tc_st8(at, o);
                            }
                        tc_wait_st();
                    }
                    named_bar_sync(1, SOFT);  // s_red is free again
                }
                // weights, row sums, e4m3 terms
                const float vinv = __int_as_float((127 - static_cast<int>(vexp)) << 23);
                uint32_t below[8];  // sign bit: in the second group
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float e = ex2(y[r] - (mref[r] == -INFINITY ? 0.0f : mref[r]));
                    l[r] = fmaf(e * vinv, e, l[r]);
                    below[r] = __float_as_uint(e - kKeySmall);
                    y[r] = e * (e < kKeySmall ? kKeyBoost * kKeyGroup : kKeyBoost) * e;
                }
                if (edge) {
                    // V rows behind the last key become zeros, and so does a NaN code that not every row sees
                    if (r0 == 0) {
                        ok = ok && ring.wait_full(ring.v_load(x), a.err, abort_flag);
                        uint8_t* v = sm + (ring.v_load(x) % SL) * S::kSlot + S::Tile::kV + S::Tile::row(tt);
                        bool nan = false;
                        if (key >= lim_max) {
#pragma unroll
                            for (int c = 0; c < S::kChunks; ++c)
                                for (int u = 0; u < CW / 16; ++u)
                                    *reinterpret_cast<uint4*>(v + c * S::Tile::kChunk + u * 16) = make_uint4(0, 0, 0, 0);
                        } else if (key >= lim_min) {
#pragma unroll
                            for (int c = 0; c < S::kChunks; ++c)
                                for (int u = 0; u < CW / 4; ++u) {
                                    uint32_t* p = reinterpret_cast<uint32_t*>(v + c * S::Tile::kChunk) + u;
                                    const uint32_t bad = e4m3_nan_mask(*p);
                                    if (bad) {
                                        *p &= ~bad;
                                        nan = true;
                                    }
                                }
                        }
                        if (nan) s_nan = 1;
                    }
                }
                uint8_t* p = s_p + x % BUFS * S::kP + tt * 16;
                uint32_t code[4][PT];
#pragma unroll
                for (int r = 0; r < 8; r += 2) e4m3_split2<PT>(y[r], y[r + 1], code[r / 2]);
                const uint32_t m0 = sign_bytes(below[0], below[1], below[2], below[3]);
                const uint32_t m1 = sign_bytes(below[4], below[5], below[6], below[7]);
                if (BUFS == 1 && i > 0 && !mbar_try_wait(&pv_done[0], phase(x - 1)))
                    ok = ok && mbar_wait_bounded(&pv_done[0], phase(x - 1), a.err, abort_flag);
#pragma unroll
                for (int b = 0; b < PT; ++b) {
                    const uint32_t c0 = code[0][b] | (code[1][b] << 16), c1 = code[2][b] | (code[3][b] << 16);
                    *reinterpret_cast<uint4*>(p + (b * RB + r0) / 8 * (kKeyTile * 16)) = make_uint4(c0 & ~m0, c1 & ~m1, c0 & m0, c1 & m1);
                }
                fence_proxy_async_smem();
                tc_fence_before();
                mbar_arrive(&p_ready[x % BUFS]);
            }
            if (left) break;
            t += nt;
            // the item's sums, then O
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const float s = warp_sum(l[r]);
                if (lane == 0) s_red[wq][r0 + r] = s;
            }
            ok = ok && mbar_wait_bounded(&pv_done[(t - 1) % BUFS], phase(t - 1), a.err, abort_flag);
            if (named_bar_or(1, SOFT, !ok)) break;
            tc_fence_after();
            const bool nan_left = s_nan;
#pragma unroll
            for (int r = 0; r < 8; ++r) l[r] = s_red[0][r0 + r] + s_red[1][r0 + r] + s_red[2][r0 + r] + s_red[3][r0 + r];
            named_bar_sync(1, SOFT);  // s_red is free again
            if (tid == 0) s_nan = 0;  // before the next item's barriers

            const long long item0 = w.tile0();  // the item's first tile in the sequence
            const bool whole = t_begin == 0 && nt == real;
            constexpr int kSlot = (RB * (D + 2) + 3) / 4 * 4;
            float* slot = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (t_begin == 0 ? 1 : 0)) * kSlot;
            // o is the result already; a row that saw no key keeps the reference -inf
            auto put = [&](int r, int d, float o, float mm, float ll) {
                if (r >= nrow) return;
                static_cast<T*>(a.out)[s_off[item & 1][r] + d] = static_cast<T>(mm == -INFINITY && ll == 0.0f ? 0.0f : o);
                if (d == 0 && a.lse) a.lse[s_lse[item & 1][r]] = ll == 0.0f ? -INFINITY : (2.0f * mm + log2f(ll)) * 0.6931471805599453f;
            };
            // Runs once per item, mostly from a cold instruction cache: one reciprocal per row (to 2
            // units of fp32 for bf16 results) and one chunk's code.
            auto reciprocal = [](float ll) { return sizeof(T) == 2 ? __fdividef(1.0f, ll) : __frcp_rn(ll); };
            float scale[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) scale[r] = reciprocal(l[r]);
#pragma unroll 1
            for (int c = 0; c < S::kChunks; ++c) {
                float o[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) o[r] = 0.0f;
#pragma unroll
                for (int b = 0; b < PT; ++b) {
                    float v[2][8];
                    tc_ld8(o_lanes + c * NP + 2 * b * RB, v[0]);
                    tc_ld8(o_lanes + c * NP + 2 * b * RB + 8, v[1]);
                    tc_wait_ld();
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        o[r] = fmaf(fmaf(v[1][r], 1.0f / kKeyGroup, v[0][r]),
                                    1.0f / (static_cast<float>(1 << (4 * b)) * kKeyBoost), o[r]);
                }
                if (nan_left && tt < CW) {  // the rows that see it have a NaN in its element
                    const int d = c * CW + tt, lo = max(lim_min, t_begin * kKeyTile), hi = min(lim_max, (t_begin + nt) * kKeyTile);
#pragma unroll 1
                    for (int k = lo; k < hi; ++k)
                        if (key_nan32(a, w.req, w.h, D, d & ~31, k, k + 1) >> (d & 31) & 1u) {
#pragma unroll
                            for (int r = 0; r < 8; ++r)
                                if (k < s_lim[r0 + r]) o[r] = __int_as_float(0x7fc00000);
                        }
                    __syncwarp();  // the loads are the whole warp's
                }
                if (tt < CW) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        if (whole) put(r0 + r, c * CW + tt, o[r] * scale[r], mref[r], l[r]);
                        else slot[(r0 + r) * D + c * CW + tt] = o[r];
                    }
                }
            }
            tc_fence_before();
            if (!whole) {
                if (tt == 0) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        slot[RB * D + r0 + r] = mref[r];
                        slot[RB * D + RB + r0 + r] = l[r];
                    }
                }
                const int c_first = key_owner(item0, s_range.total, s_range.grid);
                const int c_last = key_owner(item0 + real - 1, s_range.total, s_range.grid);
                named_bar_sync(1, SOFT);
                if (tid == 0) {
                    const unsigned parts = static_cast<unsigned>(c_last - c_first + 1);
                    const unsigned got = atom_add_acq_rel(a.counters + c_first, 1u);
                    s_last = got + 1 == parts;
                    if (s_last) a.counters[c_first] = 0;
                }
                named_bar_sync(1, SOFT);
                if (s_last) {
                    // the parts' references and sums to factors, 32 parts at a time, then O: every
                    // thread sums its float4s over the parts, eight parts' loads in flight
                    auto part_of = [&](int c) {
                        return a.part + (static_cast<size_t>(c) * 2 + (c == c_first ? 1 : 0)) * kSlot;
                    };
                    constexpr int TR = 16, kVec = D / 64;
                    const int r = tid / TR, parts = c_last - c_first + 1;
                    float mm = -INFINITY, ll = 0.0f;
                    for (int c = tid % TR; c < parts; c += TR) mm = fmaxf(mm, __ldcg(part_of(c_first + c) + RB * D + r));
#pragma unroll
                    for (int o = TR / 2; o >= 1; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
                    float4 o[kVec];
#pragma unroll
                    for (int j = 0; j < kVec; ++j) o[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int c0 = 0; c0 < parts; c0 += 32) {
                        const int nc = min(32, parts - c0);
                        for (int c = tid % TR; c < nc; c += TR) {
                            const float* p = part_of(c_first + c0 + c) + RB * D;
                            const float mc = __ldcg(p + r);
                            const float f = mc == mm ? 1.0f : exp2f(mc - mm);
                            s_fac[c][r] = f * f;
                            ll = fmaf(__ldcg(p + RB + r) * f, f, ll);
                        }
                        named_bar_sync(1, SOFT);
#pragma unroll 8
                        for (int c = 0; c < nc; ++c) {
                            const float4* p = reinterpret_cast<const float4*>(part_of(c_first + c0 + c));
#pragma unroll
                            for (int j = 0; j < kVec; ++j) {
                                const float4 x = __ldcg(p + j * SOFT + tid);
                                const float f = s_fac[c][(j * SOFT + tid) * 4 / D];
                                o[j].x = fmaf(x.x, f, o[j].x), o[j].y = fmaf(x.y, f, o[j].y);
                                o[j].z = fmaf(x.z, f, o[j].z), o[j].w = fmaf(x.w, f, o[j].w);
                            }
                        }
                        named_bar_sync(1, SOFT);
                    }
#pragma unroll
                    for (int x = TR / 2; x >= 1; x >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, x);
                    if (tid % TR == 0) {
                        s_red[0][r] = mm;
                        s_red[1][r] = ll;
                    }
                    named_bar_sync(1, SOFT);
#pragma unroll
                    for (int j = 0; j < kVec; ++j) {
                        const int e = (j * SOFT + tid) * 4, row = e / D, d = e % D;
                        const float m2 = s_red[0][row], l2 = s_red[1][row], inv = reciprocal(l2);
                        put(row, d, o[j].x * inv, m2, l2);
                        put(row, d + 1, o[j].y * inv, m2, l2);
                        put(row, d + 2, o[j].z * inv, m2, l2);
                        put(row, d + 3, o[j].w * inv, m2, l2);
                    }
                    named_bar_sync(1, SOFT);  // s_red is free again
                }
            }
            ++item;
            w.next();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        tc_dealloc(tmem, S::kCols);
    }
}

bool kv8_encode_map(const dm_kv8_cache* c, bool pair, CUtensorMap* map) {
    typedef CUresult (*Fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                           const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                           CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Fn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<Fn>(p);
    }();
    if (!fn) return false;
    const cuuint32_t cw = c->head_dim >= 128 ? 128 : 64;
    const cuuint64_t d = static_cast<cuuint64_t>(c->head_dim), chunks = d / cw, hkv = static_cast<cuuint64_t>(c->num_kv_heads);
    const cuuint64_t dims[5] = {cw, 8, chunks, 2, 4 * hkv * static_cast<cuuint64_t>(c->num_pages)};
    const cuuint64_t strides[4] = {d, cw, hkv * kKv8Page * d, 8 * d};
    const cuuint32_t box[5] = {cw, 8, static_cast<cuuint32_t>(chunks), pair ? 2u : 1u, 2}, estr[5] = {1, 1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, c->pages, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              cw == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int RB, int CTAS>
static cudaError_t launch_keys(const KeyArgs& ka, int num_sms, int dev, cudaStream_t s) {
    using S = KeyShape<T, D, RB, CTAS>;
    static std::atomic<bool> ready[64];
    if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(kv8_attn_keys_kernel<T, D, RB, CTAS>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
    }
    kv8_attn_keys_kernel<T, D, RB, CTAS><<<num_sms * S::kCtas, S::kThreads, S::kSmem, s>>>(ka);
    return cudaGetLastError();
}

// CTAs per SM.  A tile's chain of waits takes 0.65 us and more whatever D is, its bytes from HBM
// 0.37 us at D = 64 and 1.5 us at D = 256: two CTAs overlap their chains where they fit (D <= 128).
// With 16 rows two leave each thread 96 registers, with some spills.  us with two / with one, fp32 and
// bf16: D = 64, 32 requests of 2000 to 8000 keys with 3 tokens 48/56 and 48/53, of 8000 keys with one
// token of 16 heads per kv head 45/48 and 39/41; 5 chunks of up to 300 rows in fp32 156/204 (D = 128
// 359/469); D = 128, 32 requests with 3 tokens 70/70 and 61/60.  One token at D = 128 took 48 us with
// two and 45 with one, so it takes one there.
template <typename T, int RB>
static cudaError_t launch_keys_d(const KeyArgs& ka, int D, int num_sms, int dev, cudaStream_t s) {
    if (D == 64) return launch_keys<T, 64, RB, 2>(ka, num_sms, dev, s);
    if (D == 256) return launch_keys<T, 256, RB, 1>(ka, num_sms, dev, s);
    if constexpr (RB == 16)
        if (ka.a.max_q == 1) return launch_keys<T, 128, RB, 1>(ka, num_sms, dev, s);
    return launch_keys<T, 128, RB, 2>(ka, num_sms, dev, s);
}

// Rows of an item: 16 when a request's rows fill more than 8 (the cache is then read once
// for 16 rows), else 8.
cudaError_t launch_kv8_keys(const dm_kv8_cache* c, const Kv8AttnArgs& a, bool f32, int num_sms, int dev, cudaStream_t s) {
    KeyArgs ka{};
    if (!kv8_encode_map(c, true, &ka.map)) return cudaErrorNotSupported;
    ka.a = a;
    const bool wide = static_cast<int64_t>(a.max_q) * a.group > 8;
    ka.a.exact = kv8_exact(a, wide ? 16 : 8);
    if (f32) return wide ? launch_keys_d<float, 16>(ka, c->head_dim, num_sms, dev, s)
                         : launch_keys_d<float, 8>(ka, c->head_dim, num_sms, dev, s);
    return wide ? launch_keys_d<__nv_bfloat16, 16>(ka, c->head_dim, num_sms, dev, s)
                : launch_keys_d<__nv_bfloat16, 8>(ka, c->head_dim, num_sms, dev, s);
}

size_t kv8_keys_part_floats(int D, int num_sms) { return static_cast<size_t>(num_sms) * 2 * 2 * 16 * (D + 2); }

}  // namespace dm
