// dm_kv8_queries.cu — attention over the 8-bit paged cache with the queries on the tensor
// cores' M side: prompts and chunks of many bf16 query rows.
//
// Work: an item is 128 query rows (a row = one query token and one query head; the heads of a
// group share their keys, so a group's rows go together) of one request and kv head; its keys
// come in tiles of 128 tokens.  Per tile, on tcgen05 with e4m3 operands straight from the cache:
//   S [128 x 128] = (Q0 + Q1) [128 x D] . codeK^T,   O [128 x D] += (P0 + P1 + P2) [128 x 128] . codeV
// q and the weights are sums of 8-bit terms of one scale, so all products of a sum add into one
// accumulator at half the cost of a bf16 product each, and the cache needs no conversion.  bf16's 8
// bits fit two e4m3 terms: q, scaled to a largest magnitude in [2^7, 2^8) per row, is exact down to
// 2^-10 of it and off by 2^-17 of it at most.  The weights need range as well, for thousands of keys
// may lie many nats below one whose V is small: three e5m2 terms of 2^11 w (A and B need not be of
// one 8-bit type) are off by 2^-9 w down to w = 2^-19 of the reference, by 2^-28 of it below.  Two
// e4m3 terms of 2^6 w lost all below 2^-16.  fp16 weights were slower, for V's codes have to become
// fp16 too and that copy takes as much of shared memory's bandwidth as the products' operands: one
// prompt of 8192 (16 query heads on 2, D = 64 / 128 / 256) 416 / 479 / 598 us with V converted by the
// softmax warps, 368 / 473 / 681 by four more, 376 / 394 / 529 this way.
//
// Softmax as in the key-side kernel: y = x + v - M in log2 units with the page's sV = 2^v folded
// in, M raised when some y exceeds 4, o = sum w codeV / sum w 2^-v.  A row belongs to two
// threads, 64 keys of the tile each, that meet at a 64-thread barrier to agree on M; O is
// rescaled only by warps with a raised row.
//
// Roles (352 threads): 8 softmax warps (two per quarter of the rows), a producer warp, one that issues
// the scores and one that issues the O products (each is held up by the tensor cores' short queue and
// by its own waits; together they keep the queue filled).  The scores of tile x + 1 follow as soon as
// those of tile x are in registers and mostly run before the O product of tile x, so the softmax has
// the time of two products.  Between items the softmax warps turn the next item's q rows into terms
// while the last O product runs (a warp that brought those rows into L2 before gained nothing: 2.07 ms
// with it, 2.04 without for the prompts below), then write the
// item's O while the next scores run (two separate warps for the terms were slower: the
// conversions are ALU work that all four schedulers have to share).  Tensor memory: the scores
// (128 columns), two buffers of weights (96 each; at D = 256 one, written once the O product before
// is done, which it mostly is by then), O (D).  Split of the work, joins and bounded waits
// as in the key-side kernel; after a failed wait every thread runs through the remaining barriers
// without work.
//
// Bound by the softmax warps' instructions and the products together: 4 prompts of 8192 tokens,
// 16 query heads on 2 kv heads of 256, take 2.05 ms in a graph of three, 1.07 PFLOP/s or 0.64 of the
// measured bf16 rate, and 2.34 to 2.44 ms back to back under the power cap.  Two prompts of 4096: tensor
// pipe busy 54 % of the cycles, ALU 33 %, the exponential's unit 22 %.  Slower, measured with two e4m3
// terms per weight (1.95 ms): a polynomial for every fourth exponential (2.30 ms), four threads per row
// (D = 128 1.49 -> 1.60 ms), 32 columns at a time in the join (2.03 ms).
#include <atomic>
#include <cmath>
#include <type_traits>

#include "dm_kv8_walk.cuh"

namespace dm {

constexpr int kQryRows = 128;
constexpr int kQrySoft = 256;
constexpr int kQryThreads = kQrySoft + 96;  // the softmax, then three warps
// an item's start and end in tiles (KeyWalk): q rows to terms and the first scores before, O after,
// which cost this kernel as much as 6 tiles do; ranges cut by tiles alone end up to that much apart (one
// prompt of 8192 at D = 64 / 128 / 256 with 3: 374 / 430 / 715 us, 6: 387 / 397 / 524, 9: 400 / 409 / 522)
constexpr int kQryLead = 6;
// log2 units a weight may exceed the reference by: a raise makes the row wait for the O product before
// and holds up the tile (2: 426 / 432 / 577 us for the three prompts above, 3: 380 / 401 / 534, 4: 376 /
// 394 / 529, 5 the same)
constexpr float kQryLazy = 4.0f;
// log2 of what enters as a page's largest weight: below kQryTiny it is put to kQryZero, still a zero as fp16
constexpr float kQryTiny = -60.0f, kQryZero = -26.0f;
constexpr float kQryBoost = 11.0f;  // weights enter as 2^11 w <= 2^15
constexpr int kQryTerms = 3;        // e5m2 terms of a weight, 32 columns of tensor memory each

template <int D>
struct QryShape {
    static constexpr int CW = D >= 128 ? 128 : D;
    static constexpr int kChunks = D / CW;
    using Tile = KeyTile<D, false>;
    static constexpr int kTileBytes = Tile::kSlot;
    static constexpr int kTerm = kQryRows * D;  // one term of Q
    static constexpr int kFixed = 2 * kTerm + 1024;
    static constexpr int kFit = (227 * 1024 - 6144 - kFixed) / kTileBytes;
    static constexpr int kSlots = kFit > kKeyMaxSlots ? kKeyMaxSlots : kFit;
    static constexpr size_t kSmem = static_cast<size_t>(kSlots) * kTileBytes + kFixed;
    static_assert(kSlots >= 4, "shape");
};

struct QryArgs {
    CUtensorMap map;
    Kv8AttnArgs a;
};

template <int D>
__global__ void __launch_bounds__(kQryThreads, 1) kv8_attn_queries_kernel(const __grid_constant__ QryArgs qa) {
    using S = QryShape<D>;
    constexpr int CW = S::CW, SL = S::kSlots, RB = kQryRows;
    // tensor memory columns: scores, weights (two buffers, at D = 256 room for one), O
    constexpr uint32_t PB = D == 256 ? 1 : 2, kPCols = 32 * kQryTerms, kPw = 128, kO = D == 256 ? 256 : kPw + PB * kPCols;
    static_assert(kPw + PB * kPCols <= kO && kO + D <= 512, "tensor memory");
    const Kv8AttnArgs& a = qa.a;
    extern __shared__ __align__(1024) uint8_t qry_smem[];
    uint8_t* sm = qry_smem + ((1024u - (smem_u32(qry_smem) & 1023u)) & 1023u);
    uint8_t* s_q = sm + SL * S::kTileBytes;
    __shared__ __align__(8) KeyRing<SL, false> ring;
    __shared__ __align__(8) uint64_t s_full, s_free, p_ready[2], pv_done[2], q_ready, done_bar[2];
    __shared__ float s_max[2][RB], s_l[2][RB];
    __shared__ long long s_sum[64];
    __shared__ KeyRange s_range;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ int4 s_nan[2];  // by the item's parity: request, kv head and keys whose NaN codes were left out of O
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int* abort_flag = &s_abort;
    constexpr int W_LOAD = 8, W_MMA = 9;

    if (tid == 0) {
        ring.init();
        for (int i = 0; i < 2; ++i) {
            mbar_init(&p_ready[i], kQrySoft);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(&s_full, 1);
        mbar_init(&s_free, kQrySoft);
        mbar_init(&q_ready, kQrySoft);
        mbar_init(&done_bar[0], 1);
        mbar_init(&done_bar[1], 1);
        mbar_fence_init();
        s_abort = 0;
    }
    if (warp == W_MMA) tc_alloc(&s_tmem, 512);
    tc_fence_before();
    // a part of 128 rows is costly to join: four tiles per CTA at least
    const bool active = key_range<RB, kQryLead, kQryThreads>(a, 4 + kQryLead, s_sum, &s_range);
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp == W_LOAD) {
        if (active) key_produce<RB, kQryLead, D, SL, false>(a, &qa.map, sm, ring, s_range, abort_flag);
        if (a.fill) key_fill<__nv_bfloat16, D>(a);
    } else if (active && warp == W_MMA) {
        // ---------------- scores ----------------
        if (lane == 0) {
            bool ok = true;
            const uint32_t i_s = f8_idesc(128, kKeyTile, false, false);
            const uint32_t sq = smem_u32(s_q);
            KeyWalk<RB, kQryLead> w(a, s_range);
            uint32_t x = 0, item = 0;
            while (w.unit < w.end && ok) {
                int begin, last, real;
                w.span(begin, last, real);
                if (last > begin) ok = mbar_wait_bounded(&q_ready, item++ & 1u, a.err, abort_flag);
                for (; begin < last && ok; ++begin, ++x) {
                    const uint32_t ld = ring.k_load(x);
                    ok = ring.wait_full(ld, a.err, abort_flag) && mbar_wait_bounded(&s_free, (x & 1u) ^ 1u, a.err, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t k = smem_u32(sm + (ld % SL) * S::kTileBytes);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int c = 0; c < S::kChunks; ++c) {
                            const uint64_t ad = f8_desc_k<CW>(sq + t * S::kTerm + c * (RB * CW), 8 * CW);
                            const uint64_t bd = f8_desc_k<CW>(k + c * S::Tile::kChunk, S::Tile::kGroup);
#pragma unroll
                            for (int j = 0; j < CW / 32; ++j)
                                f8_mma(tmem, ad + 2 * j, bd + 2 * j, i_s, t > 0 || c > 0 || j > 0);
                        }
                    tc_commit(&s_full);
                    tc_commit(&ring.empty[ld % SL]);
                }
                w.next();
            }
            tc_commit(&done_bar[0]);
            mbar_wait_bounded(&done_bar[0], 0, a.err, nullptr);
        }
    } else if (active && warp == W_MMA + 1) {
        // ---------------- O products ----------------
        if (lane == 0) {
            bool ok = true;
            const uint32_t i_o = f8_idesc(128, D, false, true) | (1u << 7);  // A e5m2
            KeyWalk<RB, kQryLead> w(a, s_range);
            uint32_t x = 0;
            while (w.unit < w.end && ok) {
                int begin, last, real;
                w.span(begin, last, real);
                for (int i = begin; i < last && ok; ++i, ++x) {
                    const uint32_t ld = ring.v_load(x);
                    ok = ring.wait_full(ld, a.err, abort_flag) &&
                         mbar_wait_bounded(&p_ready[x & 1u], (x >> 1) & 1u, a.err, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = f8_desc_m<CW>(smem_u32(sm + (ld % SL) * S::kTileBytes), S::Tile::kChunk, S::Tile::kGroup);
                    const uint32_t p = tmem + kPw + x % PB * kPCols;
#pragma unroll
                    for (int t = 0; t < kQryTerms; ++t)
#pragma unroll
                        for (int j = 0; j < kKeyTile / 32; ++j)
                            f8_mma_ts(tmem + kO, p + t * 32 + j * 8, vd + j * (4 * S::Tile::kGroup / 16), i_o, i > begin || t > 0 || j > 0);
                    tc_commit(&pv_done[x & 1u]);
                    tc_commit(&ring.empty[ld % SL]);
                }
                w.next();
            }
            tc_commit(&done_bar[1]);
            mbar_wait_bounded(&done_bar[1], 0, a.err, nullptr);
        }
    } else if (active) {
        // ---------------- Q terms, softmax, epilogue ----------------
        const int row = tid & 127, half = tid >> 7, wq = warp & 3;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * wq) << 16);
        constexpr int H = D / 2;  // a thread's share of its row's q and O
        uint32_t t = 0, item = 0;
        bool ok = true;
        struct Done {  // an item whose O waits for its epilogue
            long long tile0;
            int64_t row;
            int t_begin, nt, real, head, lim;  // lim: keys that the row sees; -1: no row
            bool nan;
            float mref, l;
        } done;
        done.nt = 0;
        auto epilogue = [&] {
            ok = ok && mbar_wait_bounded(&pv_done[(t - 1) & 1u], ((t - 1) >> 1) & 1u, a.err, abort_flag);
            __syncwarp();
            tc_fence_after();
            const bool whole = done.t_begin == 0 && done.nt == done.real;
            const float mref = done.mref, l = done.l;
            constexpr int kSlot = RB * (D + 2);
            float* slot = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (done.t_begin == 0 ? 1 : 0)) * kSlot;
            const bool live = ok && done.lim >= 0;
            __nv_bfloat16* out =
                static_cast<__nv_bfloat16*>(a.out) + done.row * a.o_rs + static_cast<int64_t>(done.head) * a.o_hs;
            // 16 consecutive results of this row from element d on
            auto put16 = [&](const float* o, int d, float inv, bool none) {
                uint32_t wd[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(none ? 0.0f : o[2 * k] * inv, none ? 0.0f : o[2 * k + 1] * inv);
                    wd[k] = *reinterpret_cast<const uint32_t*>(&b);
                }
                if (a.o_vec) {
                    stg_v8(out + d, wd);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        out[d + 2 * k] = __ushort_as_bfloat16(static_cast<unsigned short>(wd[k]));
                        out[d + 2 * k + 1] = __ushort_as_bfloat16(static_cast<unsigned short>(wd[k] >> 16));
                    }
                }
            };
            auto put_lse = [&](float mm, float ll) {
                if (a.lse && half == 0)
                    a.lse[done.row * a.Hq + done.head] = ll == 0.0f ? -INFINITY : (mm - kQryBoost + log2f(ll)) * 0.6931471805599453f;
            };
            const float inv = 1.0f / l;
            const bool none = mref == -INFINITY && l == 0.0f;
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 32) {
                const int d = half * (D / 2) + c;
                float o[32];
                tc_ld32(lanes + kO + d, o);
                tc_wait_ld();
                if (done.nan) {  // the rows that see one have a NaN in its element
                    const int4 n = s_nan[(item - 1) & 1u];
                    const uint32_t bits = key_nan32(a, n.x, n.y, D, d, n.z, min(n.w, done.lim));
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (bits >> j & 1u) o[j] = __int_as_float(0x7fc00000);
                    __syncwarp();  // the loads are the whole warp's
                }
                if (whole) {
                    if (live) {
                        put16(o, d, inv, none);
                        put16(o + 16, d + 16, inv, none);
                    }
                } else if (ok) {
                    // element-major, so that a warp's stores are contiguous
#pragma unroll
                    for (int j = 0; j < 32; ++j) slot[(d + j) * RB + row] = o[j];
                }
            }
            tc_fence_before();
            if (whole) {
                if (live) put_lse(mref, l);
            } else {
                if (half == 0 && ok) {
                    slot[RB * D + row] = mref;
                    slot[RB * D + RB + row] = l;
                }
                const int c_first = key_owner(done.tile0, s_range.total, s_range.grid),
                          c_last = key_owner(done.tile0 + done.real - 1, s_range.total, s_range.grid);
                if (!named_bar_or(1, kQrySoft, !ok)) {
                    if (tid == 0) {
                        const unsigned got = atom_add_acq_rel(a.counters + c_first, 1u);
                        s_last = got + 1 == static_cast<unsigned>(c_last - c_first + 1);
                        if (s_last) a.counters[c_first] = 0;
                    }
                    named_bar_sync(1, kQrySoft);
                    if (s_last) {
                        auto part_of = [&](int c) {
                            return a.part + (static_cast<size_t>(c) * 2 + (c == c_first ? 1 : 0)) * kSlot;
                        };
                        float mm = -INFINITY, ll = 0.0f;
                        for (int c = c_first; c <= c_last; ++c) mm = fmaxf(mm, __ldcg(part_of(c) + RB * D + row));
                        for (int c = c_first; c <= c_last; ++c) {
                            const float* p = part_of(c) + RB * D + row;
                            const float mc = __ldcg(p), f = mc == mm ? 1.0f : exp2f(0.5f * (mc - mm));
                            ll = fmaf(__ldcg(p + RB) * f, f, ll);
                        }
                        const float linv = 1.0f / ll;
#pragma unroll 1
                        for (int d = half * (D / 2); d < (half + 1) * (D / 2); d += 16) {
                            float o[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = 0.0f;
                            for (int c = c_first; c <= c_last; ++c) {
                                const float* p = part_of(c);
                                const float mc = __ldcg(p + RB * D + row);
                                const float fc = mc == mm ? 1.0f : exp2f(mc - mm);
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] = fmaf(__ldcg(p + (d + j) * RB + row), fc, o[j]);
                            }
                            if (live) put16(o, d, linv, mm == -INFINITY && ll == 0.0f);
                        }
                        if (live) put_lse(mm, ll);
                    }
                }
            }
        };
        KeyWalk<RB, kQryLead> w(a, s_range);
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
            const int f = w.block() * RB + min(row, nrow - 1), tok = f / a.group, head = w.h * a.group + f % a.group;
            const int lim = row < nrow ? min(w.r.len, max(0, w.r.full - w.r.m + tok + 1)) : 0;
            float frow;
            {   // this half of the row: exact scaling to a largest magnitude in [2^7, 2^8), two terms
                const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) +
                                         static_cast<int64_t>(w.r.row0 + tok) * a.q_rs + static_cast<int64_t>(head) * a.q_hs +
                                         half * H;
                uint32_t x[H / 2];
                if (a.q_vec) {
#pragma unroll
                    for (int c = 0; c < H / 2; c += 8) ldg_v8(x + c, q + 2 * c);
                } else {
#pragma unroll
                    for (int c = 0; c < H / 2; ++c)
                        x[c] = __bfloat16_as_ushort(q[2 * c]) | static_cast<uint32_t>(__bfloat16_as_ushort(q[2 * c + 1])) << 16;
                }
                uint32_t top = 0;  // two largest magnitudes, NaN kept
#pragma unroll
                for (int c = 0; c < H / 2; ++c) top = bf16x2_max_nan(top, x[c] & 0x7fff7fffu);
                float amax = bf16lo(top) <= 3.402823466e38f && bf16hi(top) <= 3.402823466e38f ? fmaxf(bf16lo(top), bf16hi(top))
                                                                                             : INFINITY;
                s_max[half][row] = amax;
                named_bar_sync(2 + wq, 64);
                amax = fmaxf(s_max[0][row], s_max[1][row]);
                named_bar_sync(2 + wq, 64);
                const int ex = max(-120, min(120, (__float_as_int(amax) >> 23) - 127 - 7));
                frow = a.scale_log2 * __int_as_float((127 + ex) << 23);
                // a row with NaN or Inf becomes NaN, a row behind the last zero
                const float mul = row >= nrow ? 0.0f : amax == INFINITY ? __int_as_float(0x7fc00000) : __int_as_float((127 - ex) << 23);
#pragma unroll
                for (int u = 0; u < H / 16; ++u) {  // 16 elements: one 16-byte unit of each term
                    uint32_t t0[8], t1[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        e4m3_terms2(bf16lo(x[u * 8 + j]) * mul, bf16hi(x[u * 8 + j]) * mul, t0[j], t1[j]);
                    const int d = half * H + u * 16;
                    uint8_t* dst = s_q + (d / CW) * (RB * CW) + f8_unit<CW>(row, (d % CW) / 16);
                    *reinterpret_cast<uint4*>(dst) = make_uint4(t0[0] | (t0[1] << 16), t0[2] | (t0[3] << 16),
                                                                t0[4] | (t0[5] << 16), t0[6] | (t0[7] << 16));
                    *reinterpret_cast<uint4*>(dst + S::kTerm) = make_uint4(t1[0] | (t1[1] << 16), t1[2] | (t1[3] << 16),
                                                                           t1[4] | (t1[5] << 16), t1[6] | (t1[7] << 16));
                }
                fence_proxy_async_smem();
                mbar_arrive(&q_ready);
            }
            if (done.nt) epilogue();
            float mref = -INFINITY, l = 0.0f;
            bool nan_row = false;

            for (int i = 0; i < nt; ++i) {
                const uint32_t x = t + i, pb = kPw + x % PB * kPCols + half * 16;
                const int tile0 = (t_begin + i) * kKeyTile;
                const bool t1 = ring.try_meta(x);
                const bool t2 = mbar_try_wait(&s_full, x & 1u);
                const bool t3 = PB == 1 || i < 2 || mbar_try_wait(&pv_done[x & 1u], ((x - 2) >> 1) & 1u);
                if (ok && !(t1 && t2 && t3))
                    ok = ring.wait_meta(x, a.err, abort_flag) &&
                         mbar_wait_bounded(&s_full, x & 1u, a.err, abort_flag) &&
                         (PB == 1 || i < 2 || mbar_wait_bounded(&pv_done[x & 1u], ((x - 2) >> 1) & 1u, a.err, abort_flag));
                __syncwarp();
                tc_fence_after();
                float s[64];
                tc_ld32(lanes + half * 64, s);
                tc_ld32(lanes + half * 64 + 32, s + 32);
                // the half's pages: y = s f + g
                float f[4], g[4], vinv[4];
                const float base = mref == -INFINITY ? 0.0f : kQryBoost - mref;
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float2 sc = ring.meta[x % ring.kMeta][half * 4 + p];
                    const int ve = ((__float_as_int(sc.y) >> 23) & 0xff) - 127;
                    f[p] = frow * sc.x;
                    g[p] = sc.y < 0.0f ? -INFINITY : static_cast<float>(ve) + base;
                    vinv[p] = __int_as_float((127 - ve) << 23);
                }
                tc_wait_ld();
                tc_fence_before();
                mbar_arrive(&s_free);
                const bool edge = tile0 + kKeyTile > lim_min;
#pragma unroll
                for (int c = 0; c < 64; ++c) s[c] = fmaf(s[c], f[c / 16], g[c / 16]);
                // keys that the row does not see, or that lie on no page
                const bool gone = g[0] == -INFINITY || g[1] == -INFINITY || g[2] == -INFINITY || g[3] == -INFINITY;
                if (edge || gone) {
                    const int seen = lim - tile0 - half * 64;
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if (c >= seen || g[c / 16] == -INFINITY) s[c] = -INFINITY;
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // of each page
#pragma unroll
                for (int c = 0; c < 16; c += 2)
#pragma unroll
                    for (int p = 0; p < 4; ++p) m4[p] = fmaxf(m4[p], fmaxf(s[p * 16 + c], s[p * 16 + c + 1]));
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                bool low = fminf(fminf(m4[0], m4[1]), fminf(m4[2], m4[3])) < kQryTiny;
                if (edge || gone) {  // pages without a visible key are not meant
                    low = false;
#pragma unroll
                    for (int p = 0; p < 4; ++p) low = low || (m4[p] < kQryTiny && m4[p] > -INFINITY);
                }
                const bool over = mref == -INFINITY ? mx > -INFINITY : mx > kQryBoost + kQryLazy;
                if (named_bar_or(2 + wq, 64, over || low)) {
                    // the row's two threads agree on its reference; O of the raised rows follows
                    s_max[half][row] = mx;
                    named_bar_sync(2 + wq, 64);
                    const float both = fmaxf(s_max[0][row], s_max[1][row]);  // in units of the old reference
                    named_bar_sync(2 + wq, 64);
                    const bool raise = mref == -INFINITY ? both > -INFINITY : both > kQryBoost + kQryLazy;
                    float fac = 1.0f, shift = 0.0f;
                    if (raise) {
                        const float nm = mref == -INFINITY ? both : both - kQryBoost + mref;
                        shift = mref == -INFINITY ? kQryBoost - nm : mref - nm;
                        // in two factors, for the sum holds 2^-v: it may have to go down by more than one reaches
                        const float f = mref == -INFINITY ? 0.0f : exp2f(0.5f * shift);
                        mref = nm;
                        l = l * f * f;
                        fac = f * f;
                    }
                    if (raise || low) {
                        // A page whose weights are all near or below ex2's last step may still have its share of
                        // the sum, where V's scales are far apart, as pages of zeros do (their scale is 2^-100).
                        // Its scores go up, to where the weights' terms are still zero, and its 2^-v goes down
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            const float m = m4[p] + shift;
                            float up = shift;
                            if (m < kQryTiny && m > -INFINITY) {
                                const float d = fminf(floorf(kQryZero - m), 226.0f);
                                up += d;
                                vinv[p] = __int_as_float(max(0, (__float_as_int(vinv[p]) >> 23) - static_cast<int>(d)) << 23);
                            }
#pragma unroll
                            for (int c = 0; c < 16; ++c) s[p * 16 + c] += up;
                        }
                    }
                    if (__any_sync(0xffffffffu, raise) && i > 0) {
                        ok = ok && mbar_wait_bounded(&pv_done[(x - 1) & 1u], ((x - 1) >> 1) & 1u, a.err, abort_flag);
                        __syncwarp();
                        tc_fence_after();
                        // each of the two threads rescales one half of the row's O
#pragma unroll 1
                        for (int c = 0; c < D / 2; c += 32) {
                            float o[32];
                            tc_ld32(lanes + kO + half * (D / 2) + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] *= fac;
                            tc_st32(lanes + kO + half * (D / 2) + c, o);
                        }
                        tc_wait_st();
                    }
                }
                // weights, sums, terms: this half's 64 keys, columns of P0, P1 and P2
                // (of one buffer: stored together once the O product of the tile before has read its own)
                uint32_t pt[kQryTerms][PB == 1 ? 16 : 4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        float* y = s + p * 16 + c;
                        uint32_t four[kQryTerms];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            y[j] = ex2(y[j]);
                            sum[j] += y[j];
                        }
                        e5m2_terms3(y[0], y[1], y[2], y[3], four);
#pragma unroll
                        for (int t = 0; t < kQryTerms; ++t) pt[t][(PB == 1 ? p * 4 : 0) + c / 4] = four[t];
                    }
                    l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), vinv[p], l);
                    if constexpr (PB == 2) {
#pragma unroll
                        for (int t = 0; t < kQryTerms; ++t) tc_st4(lanes + pb + t * 32 + p * 4, pt[t]);
                    }
                }
                if constexpr (PB == 1) {
                    if (i > 0) {
                        if (ok && !mbar_try_wait(&pv_done[(x - 1) & 1u], ((x - 1) >> 1) & 1u))
                            ok = mbar_wait_bounded(&pv_done[(x - 1) & 1u], ((x - 1) >> 1) & 1u, a.err, abort_flag);
                        __syncwarp();
                        tc_fence_after();
                    }
#pragma unroll
                    for (int t = 0; t < kQryTerms; ++t) tc_st16(lanes + pb + t * 32, pt[t]);
                }
                if (edge) {
                    // V rows behind the last key become zeros, and so does a NaN code that not every row sees
                    if (half == 0) {
                        ok = ok && ring.wait_full(ring.v_load(x), a.err, abort_flag);
                        uint8_t* v = sm + (ring.v_load(x) % SL) * S::kTileBytes + S::Tile::row(row);
                        const int key = tile0 + row;
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
                        fence_proxy_async_smem();
                        nan_row = nan_row || nan;
                    }
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&p_ready[x & 1u]);
            }
            t += nt;
            // both halves' sums
            s_l[half][row] = l;
            named_bar_sync(2 + wq, 64);
            done.l = s_l[0][row] + s_l[1][row];
            named_bar_sync(2 + wq, 64);
            done.mref = mref;
            done.tile0 = w.tile0();
            done.row = w.r.row0 + tok;
            done.head = head;
            done.lim = row < nrow ? lim : -1;
            done.nan = false;
            if (t_end * kKeyTile > lim_min) {  // tiles that not every row sees
                if (tid == 0)
                    s_nan[item & 1u] = make_int4(w.req, w.h, max(lim_min, t_begin * kKeyTile), min(lim_max, t_end * kKeyTile));
                done.nan = named_bar_or(1, kQrySoft, nan_row);
            }
            ++item;
            done.t_begin = t_begin, done.nt = nt, done.real = real;
            w.next();
        }
        if (done.nt) epilogue();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        tc_dealloc(tmem, 512);
    }
}

template <int D>
static cudaError_t launch_queries(const QryArgs& qa, int num_sms, int dev, cudaStream_t s) {
    using S = QryShape<D>;
    static std::atomic<bool> ready[64];
    if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(kv8_attn_queries_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
    }
    kv8_attn_queries_kernel<D><<<num_sms, kQryThreads, S::kSmem, s>>>(qa);
    return cudaGetLastError();
}

cudaError_t launch_kv8_queries(const dm_kv8_cache* c, const Kv8AttnArgs& a, int num_sms, int dev, cudaStream_t s) {
    QryArgs qa{};
    if (!kv8_encode_map(c, false, &qa.map)) return cudaErrorNotSupported;
    qa.a = a;
    qa.a.exact = kv8_exact(a, kQryRows);
    if (c->head_dim == 64) return launch_queries<64>(qa, num_sms, dev, s);
    if (c->head_dim == 128) return launch_queries<128>(qa, num_sms, dev, s);
    return launch_queries<256>(qa, num_sms, dev, s);
}

size_t kv8_queries_part_floats(int D, int num_sms) { return static_cast<size_t>(num_sms) * 2 * kQryRows * (D + 2); }

}  // namespace dm
