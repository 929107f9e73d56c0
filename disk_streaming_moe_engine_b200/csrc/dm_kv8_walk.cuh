// dm_kv8_walk.cuh — what the attention kernels over the 8-bit cache share: the sequence of
// (request, row block, kv head, key tile), its cut into one range per CTA, and the producer that
// brings a range's key tiles into shared memory.
#pragma once
#include "dm_kv8_tc.cuh"

namespace dm {

constexpr int kKeyTile = 128;  // keys of a tile
constexpr int kKeyPages = kKeyTile / kKv8Page;

// What a role knows of the request it is at.
struct KeyReq {
    int row0, m, len, full, blocks, tiles;
};

struct KeyRaw {  // a request's words as loaded
    int c0, c1, len;
};
DM_DEV KeyRaw key_raw(const Kv8AttnArgs& a, int i) {
    KeyRaw w = {i, i + 1, 0};
    if (i >= a.n) return w;
    if (a.cu_q) w.c0 = a.cu_q[i], w.c1 = a.cu_q[i + 1];
    w.len = a.seq_lens[i];
    return w;
}

template <int RB>
DM_DEV KeyReq key_req(const Kv8AttnArgs& a, const KeyRaw& w, bool report) {
    KeyReq r;
    r.row0 = w.c0;
    const long long m = static_cast<long long>(w.c1) - w.c0;
    if (w.c0 < 0 || m < 0 || m > a.max_q || w.c0 + m > a.rows) {
        if (report) raise_error(a.err, DM_DEVERR_RANGE);
        r.m = 0;
    } else {
        r.m = static_cast<int>(m);
    }
    r.full = w.len;
    if (r.full < 0) {
        if (report) raise_error(a.err, DM_DEVERR_RANGE);
        r.full = 0;
    }
    r.len = r.full;
    if (r.len > a.width * kKv8Page) {
        if (report) raise_error(a.err, DM_DEVERR_CAPACITY);
        r.len = a.width * kKv8Page;
    }
    r.blocks = static_cast<int>((static_cast<long long>(r.m) * a.group + RB - 1) / RB);
    r.tiles = max(1, (r.len + kKeyTile - 1) / kKeyTile);
    return r;
}

constexpr int kKeyFew = 64;  // requests whose words a CTA keeps in shared memory

struct KeyRange {  // a CTA's range of the sequence [u0, u1), and where it starts
    long long u0, u1, total, rem;
    long long grid;
    int req, blk;
    KeyRaw raw[kKeyFew];
    DM_DEV KeyRaw request(const Kv8AttnArgs& a, int i) const {
        if (a.n <= kKeyFew && i < a.n) return raw[i];
        return key_raw(a, i);
    }
};

// keys that a block's rows see: every row those before lo, its last token's rows those before hi
template <int RB>
DM_DEV void key_limits(const Kv8AttnArgs& a, const KeyReq& r, int blk, int& lo, int& hi) {
    const int rows = r.m * a.group;
    const int first = blk * RB / a.group, last = (min(rows, (blk + 1) * RB) - 1) / a.group;
    lo = min(r.len, max(0, r.full - r.m + first + 1));
    hi = min(r.len, max(0, r.full - r.m + last + 1));
}

// Tiles that a block's rows see (an item without keys has one, so that its rows are written).
template <int RB>
DM_DEV int key_tiles(const Kv8AttnArgs& a, const KeyReq& r, int blk) {
    int lo, hi;
    key_limits<RB>(a, r, blk, lo, hi);
    return max(1, (hi + kKeyTile - 1) / kKeyTile);
}

// Position in the sequence of all items: request, then row block, kv head.  An item has LEAD
// units for its start and end and one per tile; the CTA whose range holds a tile's unit works on
// it.  exact: a block has the tiles that its rows see.  Else every block has those of the
// request's whole length (what its rows do not see is skipped) and the blocks come as first,
// last, second, second to last, ...: under a causal mask neighbours then cost the same together.
template <int RB, int LEAD>
struct KeyWalk {
    const Kv8AttnArgs& a;
    const KeyRange& range;
    long long unit, end;  // this CTA's range
    int req, blk, h, pos, tiles;
    KeyReq r;
    KeyRaw ahead;  // of request req + 1, loaded before it is needed
    DM_DEV KeyWalk(const Kv8AttnArgs& args, const KeyRange& k)
        : a(args), range(k), unit(k.u0), end(k.u1), req(k.req), blk(k.blk) {
        r = key_req<RB>(a, range.request(a, req), false);
        ahead = range.request(a, req + 1);
        tiles = a.exact ? key_tiles<RB>(a, r, blk) : r.tiles;
        const unsigned per = tiles + LEAD;
        h = k.rem >> 32 ? static_cast<int>(k.rem / per) : static_cast<int>(static_cast<unsigned>(k.rem) / per);
        pos = static_cast<int>(k.rem - static_cast<long long>(h) * per);
    }
    DM_DEV int block() const { return a.exact ? blk : blk & 1 ? r.blocks - 1 - (blk >> 1) : blk >> 1; }
    DM_DEV int count() const { return static_cast<int>(min(static_cast<long long>(tiles + LEAD - pos), end - unit)); }
    // this CTA's tiles of the item: [first, last) of the `real` ones that its rows see
    DM_DEV void span(int& first, int& last, int& real) const {
        real = a.exact ? tiles : key_tiles<RB>(a, r, block());
        first = max(0, pos - LEAD);
        last = min(real, max(0, pos + count() - LEAD));
    }
    DM_DEV long long tile0() const { return unit - pos + LEAD; }  // the unit of the item's first tile
    DM_DEV void next() {
        unit += count();
        if (unit >= end) return;
        pos = 0;
        if (++h < a.Hkv) return;
        h = 0;
        if (++blk >= r.blocks) {
            blk = 0;
            do {
                if (++req >= a.n) {  // only if the lengths changed under the kernel
                    end = unit;
                    return;
                }
                r = key_req<RB>(a, ahead, false);
                ahead = range.request(a, req + 1);
            } while (r.blocks == 0);
        }
        tiles = a.exact ? key_tiles<RB>(a, r, blk) : r.tiles;
    }
};

template <typename V>
DM_DEV V warp_scan(V v) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += y;
    }
    return v;
}

// This CTA's range of the sequence and where it starts.  At most one CTA per `min_units` units
// takes part; false: this one does not.  Up to 64 requests: a warp per request, a lane per
// block; more: a thread per share of the requests (whose blocks are few where `exact` is set).
// Called by all NT threads with s_sum [kKeyFew]; ends with a barrier.
template <int RB, int LEAD, int NT>
DM_DEV bool key_range(const Kv8AttnArgs& a, int min_units, long long* s_sum, KeyRange* out) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool report = blockIdx.x == 0;
    long long total, u0 = 0;
    bool active;
    auto cut = [&] {
        const long long grid = min(static_cast<long long>(gridDim.x), (total + min_units - 1) / min_units);
        active = blockIdx.x < grid;
        u0 = active ? total * blockIdx.x / grid : 0;
        if (tid == 0) {
            out->total = total;
            out->grid = grid;
            out->u0 = u0;
            out->u1 = active ? total * (blockIdx.x + 1) / grid : 0;
        }
    };
    if (a.n <= kKeyFew && !a.exact) {  // every warp for itself, two requests per lane
        const KeyRaw w0 = key_raw(a, lane), w1 = key_raw(a, lane + 32);
        auto units = [&](int i, const KeyRaw& w) {
            const KeyReq r = key_req<RB>(a, w, report && warp == 0 && i < a.n);
            return i < a.n ? static_cast<long long>(r.blocks) * a.Hkv * (r.tiles + LEAD) : 0;
        };
        const long long v0 = units(lane, w0), v1 = units(lane + 32, w1);
        const long long e0 = warp_scan(v0), e1 = __shfl_sync(0xffffffffu, e0, 31) + warp_scan(v1);
        total = __shfl_sync(0xffffffffu, e1, 31);
        cut();
        if (warp == 0) {
            if (lane < a.n) out->raw[lane] = w0;
            if (lane + 32 < a.n) out->raw[lane + 32] = w1;
            const bool here0 = u0 >= e0 - v0 && u0 < e0, here1 = u0 >= e1 - v1 && u0 < e1;
            if (active && (here0 || here1)) {
                const long long rem = u0 - (here0 ? e0 - v0 : e1 - v1);
                const KeyReq r = key_req<RB>(a, here0 ? w0 : w1, false);
                const long long c = static_cast<long long>(r.tiles + LEAD) * a.Hkv;
                out->req = here0 ? lane : lane + 32;
                out->blk = r.blocks > 1 ? static_cast<int>(rem / c) : 0;
                out->rem = rem - out->blk * c;
            }
        }
    } else if (a.n <= kKeyFew) {
        if (tid < a.n) {
            out->raw[tid] = key_raw(a, tid);
            key_req<RB>(a, out->raw[tid], report);
        }
        __syncthreads();
        for (int i = warp; i < a.n; i += NT / 32) {
            const KeyReq r = key_req<RB>(a, out->raw[i], false);
            long long sum = 0;
            for (int b = lane; b < r.blocks; b += 32) sum += key_tiles<RB>(a, r, b) + LEAD;
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) s_sum[i] = sum * a.Hkv;
        }
        __syncthreads();
        const long long v0 = lane < a.n ? s_sum[lane] : 0, v1 = lane + 32 < a.n ? s_sum[lane + 32] : 0;
        const long long e0 = warp_scan(v0), t0 = __shfl_sync(0xffffffffu, e0, 31), e1 = t0 + warp_scan(v1);
        total = __shfl_sync(0xffffffffu, e1, 31);
        cut();
        if (active && warp == 0) {
            const unsigned m0 = __ballot_sync(0xffffffffu, u0 >= e0 - v0 && u0 < e0);
            const unsigned m1 = __ballot_sync(0xffffffffu, u0 >= e1 - v1 && u0 < e1);
            const int src = m0 ? __ffs(m0) - 1 : __ffs(m1) - 1;
            const int req = m0 ? src : src + 32;
            long long rem = u0 - (m0 ? __shfl_sync(0xffffffffu, e0 - v0, src) : __shfl_sync(0xffffffffu, e1 - v1, src));
            const KeyReq r = key_req<RB>(a, out->raw[req], false);
            int blk = 0;
            for (;; blk += 32) {  // 32 blocks at a time
                const long long c =
                    blk + lane < r.blocks ? static_cast<long long>(key_tiles<RB>(a, r, blk + lane) + LEAD) * a.Hkv : 0;
                const long long e = warp_scan(c), all = __shfl_sync(0xffffffffu, e, 31);
                if (rem >= all && blk + 32 < r.blocks) {
                    rem -= all;
                    continue;
                }
                const unsigned m = __ballot_sync(0xffffffffu, rem < e);
                const int at = m ? __ffs(m) - 1 : 0;
                rem -= __shfl_sync(0xffffffffu, e - c, at);
                blk += at;
                break;
            }
            if (lane == 0) {
                out->req = req;
                out->blk = blk;
                out->rem = rem;
            }
        }
    } else {
        const int per = (a.n + NT - 1) / NT;
        const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
        auto blocks_of = [&](int i, bool rep, auto&& each) {  // each(block, its units over the kv heads, ...) until true
            const KeyReq r = key_req<RB>(a, key_raw(a, i), rep);
            for (int b = 0; b < r.blocks; ++b) {
                if (!a.exact) {  // all at once
                    const long long c = static_cast<long long>(r.tiles + LEAD) * a.Hkv;
                    return each(0, c * r.blocks, c);
                }
                const long long c = static_cast<long long>(key_tiles<RB>(a, r, b) + LEAD) * a.Hkv;
                if (each(b, c, c)) return true;
            }
            return false;
        };
        long long mine = 0;
        for (int i = i0; i < i1; ++i)
            blocks_of(i, report, [&](int, long long c, long long) {
                mine += c;
                return false;
            });
        long long pre = warp_scan(mine);
        if (lane == 31) s_sum[warp] = pre;
        __syncthreads();
        total = 0;
        for (int w = 0; w < NT / 32; ++w) {
            if (w == warp) pre += total - mine;  // tiles before this thread's requests
            total += s_sum[w];
        }
        cut();
        if (active && u0 >= pre && u0 < pre + mine) {
            long long at = pre;
            for (int i = i0; i < i1; ++i)
                if (blocks_of(i, false, [&](int b, long long c, long long one) {
                        if (u0 >= at + c) {
                            at += c;
                            return false;
                        }
                        const long long skip = (u0 - at) / one;
                        out->req = i;
                        out->blk = b + static_cast<int>(skip);
                        out->rem = u0 - at - skip * one;
                        return true;
                    }))
                    break;
        }
    }
    __syncthreads();
    return active;
}

// Bits of which of 32 elements from d on have a NaN code in V of some key in [lo, hi).  For keys that
// not every row of an item sees (their NaN codes are zeros in the product): read from the cache, out
// of line, for it hardly ever runs.
static __device__ __noinline__ uint32_t key_nan32(const Kv8AttnArgs& a, int req, int h, int D, int d, int lo, int hi) {
    uint32_t bits = 0;
    for (int key = lo; key < hi; ++key) {
        const int id = a.table[static_cast<size_t>(req) * a.width + key / kKv8Page];
        if (id < 0 || id >= a.num_pages) continue;
        const size_t at = ((static_cast<size_t>(id) * 2 + 1) * a.Hkv + h) * (kKv8Page * D) + static_cast<size_t>(key % kKv8Page) * D + d;
        const uint32_t* p = reinterpret_cast<const uint32_t*>(a.pages + at);
        for (int i = 0; i < 8; ++i) bits |= ((e4m3_nan_mask(p[i]) & 0x01010101u) * 0x01020408u >> 24) << (4 * i);
    }
    return bits;
}

// DM_KV8_FILL_ROWS: zeros in the rows of `out` that no request writes: those before cu_q[0] and from
// cu_q[n] on, and those of requests that are skipped.  By one warp of every CTA; out of line, for the
// instruction cache is what the prompts' kernel has least of (inlined: 4 x 8192 2.05 -> 2.20 ms).
template <typename T, int D>
__device__ __noinline__ void key_fill(const Kv8AttnArgs& a) {
    constexpr int EV = 16 / sizeof(T);  // elements of 16 bytes
    const int lane = threadIdx.x & 31;
    auto clip = [&](long long r) { return static_cast<int>(min(max(r, 0ll), static_cast<long long>(a.rows))); };
    auto row = [&](int r) {
        for (int i = lane; i < a.Hq * (D / EV); i += 32) {
            T* o = static_cast<T*>(a.out) + static_cast<int64_t>(r) * a.o_rs + static_cast<int64_t>(i / (D / EV)) * a.o_hs + i % (D / EV) * EV;
            if (a.o_vec) {
                *reinterpret_cast<uint4*>(o) = make_uint4(0, 0, 0, 0);
            } else {
                for (int e = 0; e < EV; ++e) o[e] = static_cast<T>(0.0f);
            }
        }
    };
    auto shared_rows = [&](long long lo, long long hi) {  // by all CTAs together
        const int end = clip(hi);
        for (long long r = clip(lo) + static_cast<long long>(blockIdx.x); r < end; r += gridDim.x) row(static_cast<int>(r));
    };
    if (a.cu_q) shared_rows(0, a.cu_q[0]);
    shared_rows(a.cu_q ? a.cu_q[a.n] : a.n, a.rows);
    for (long long base = static_cast<long long>(blockIdx.x) * 32; a.cu_q && base < a.n; base += static_cast<long long>(gridDim.x) * 32) {
        const int i = static_cast<int>(min(base + lane, static_cast<long long>(a.n)));
        long long c0 = 0, c1 = 0;
        if (i < a.n) c0 = a.cu_q[i], c1 = a.cu_q[i + 1];
        unsigned skipped = __ballot_sync(0xffffffffu, c1 > c0 && (c0 < 0 || c1 - c0 > a.max_q || c1 > a.rows));
        while (skipped) {
            const int l = __ffs(skipped) - 1;
            skipped &= skipped - 1;
            const int end = clip(__shfl_sync(0xffffffffu, c1, l));
            for (int r = clip(__shfl_sync(0xffffffffu, c0, l)); r < end; ++r) row(r);
        }
    }
}

// The CTA whose range holds unit u.
DM_DEV int key_owner(long long u, long long total, long long grid) { return static_cast<int>(((u + 1) * grid - 1) / total); }

// Shared memory of the key tiles: a ring of SL slots.  PAIR: a slot takes a tile's K and V and is
// free again after its O product.  Else a slot takes K or V of one tile, loaded in the order K0,
// K1, V0, K2, V1, ..., and is free as soon as the one product that reads it is done: the ring then
// holds what the next products need.  The query-side kernel is bound by its products and by how
// early the next tile is there (4 x 8192 prompts 3.24 ms in pairs, 2.73 ms single); the key-side
// one by the bytes (64 x 32768 384 us in pairs, 405 us single).
constexpr int kKeyMaxSlots = 12;

template <int SL, bool PAIR>
struct KeyRing {
    // Tiles whose scales are kept.  Those of tile x + kMeta are written once its K has a slot, i.e.
    // the K or O product of the tile SL positions before is done; by then every softmax thread has
    // left tile x: in pairs that was the O product of tile x itself, else the scores of tile x + 2
    // (issued after the weights of tile x) or a later O product.
    static constexpr int kMeta = PAIR ? SL : SL / 2 + 2;
    uint64_t full[SL], empty[SL], meta_full[kMeta];
    float2 meta[kMeta][kKeyPages];  // (sK, sV) of the tile's pages; sV < 0: no such page
    static DM_DEV uint32_t k_load(uint32_t tile) { return PAIR ? tile : tile ? 2 * tile - 1 : 0; }
    static DM_DEV uint32_t v_load(uint32_t tile) { return PAIR ? tile : 2 * tile + 2; }
    DM_DEV void init() {               // one thread
        for (int i = 0; i < SL; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < kMeta; ++i) mbar_init(&meta_full[i], 1);
    }
    DM_DEV bool wait_full(uint32_t load, uint32_t* err, volatile int* abort_flag) {
        return mbar_wait_bounded(&full[load % SL], (load / SL) & 1u, err, abort_flag);
    }
    // scales of tile x: ready (or not yet)
    DM_DEV bool try_meta(uint32_t x) { return mbar_try_wait(&meta_full[x % kMeta], (x / kMeta) & 1u); }
    DM_DEV bool wait_meta(uint32_t x, uint32_t* err, volatile int* abort_flag) {
        return mbar_wait_bounded(&meta_full[x % kMeta], (x / kMeta) & 1u, err, abort_flag);
    }
};

// Where a tile's bytes lie in its slot: blocks of 8 tokens, in each K then V (in pairs), in each
// the head's chunks of 8 rows x CW bytes.
template <int D, bool PAIR>
struct KeyTile {
    static constexpr int CW = D >= 128 ? 128 : D, kChunks = D / CW;
    static constexpr int kChunk = 8 * CW;                          // from chunk to chunk
    static constexpr int kGroup = (PAIR ? 2 : 1) * kChunks * kChunk;  // from block to block
    static constexpr int kV = PAIR ? kChunks * kChunk : 0;         // V behind K
    static constexpr int kSlot = kKeyTile / 8 * kGroup;
    static DM_DEV int row(int token) { return token / 8 * kGroup + token % 8 * CW; }  // chunk 0
};

// Producer (one warp): a tile's K or V (or both) in one TMA box per page, one lane per page; page
// ids fetched two groups of 4 tiles ahead of their use, scales one group ahead.  A page that is
// missing or holds no key of the item reads zeros.
template <int RB, int LEAD, int D, int SL, bool PAIR>
DM_DEV void key_produce(const Kv8AttnArgs& a, const CUtensorMap* map, uint8_t* sm, KeyRing<SL, PAIR>& ring,
                        const KeyRange& range, volatile int* abort_flag) {
    using Tile = KeyTile<D, PAIR>;
    constexpr int kSlot = Tile::kSlot;
    const int lane = threadIdx.x & 31;
    bool ok = true;
    KeyWalk<RB, LEAD> w(a, range);
    int ti = -1, ei = 0, hi = 0;  // next tile of w's item, end of its tiles, its keys
    struct Group {
        int count = 0;             // tiles
        int id = -1, h = 0;        // this lane's page (tile lane / 8, page lane % 8) and kv head
        bool wanted = false;       // a key of the item lies on it
        float2 sc = make_float2(0.0f, -1.0f);
    };
    auto fetch_ids = [&](Group& g) {
        g = Group();
        while (g.count < 32 / kKeyPages && w.unit < w.end) {
            if (ti < 0) {
                int lo, real;
                key_limits<RB>(a, w.r, w.block(), lo, hi);
                w.span(ti, ei, real);
            }
            if (ti < ei) {
                const int p = ti * kKeyPages + lane % kKeyPages;
                if (lane / kKeyPages == g.count) {
                    g.h = w.h;
                    g.wanted = p * kKv8Page < hi;
                    if (g.wanted) g.id = a.table[static_cast<size_t>(w.req) * a.width + p];
                }
                ++g.count;
                ++ti;
            } else {
                w.next();
                ti = -1;
            }
        }
    };
    auto fetch_scales = [&](Group& g) {
        if (!g.wanted) return;
        if (g.id >= 0 && g.id < a.num_pages) {
            const float* sc = a.scales + static_cast<size_t>(g.id) * 2 * a.Hkv + g.h;
            g.sc = make_float2(sc[0], sc[a.Hkv]);
        } else {
            g.id = -1;
            raise_error(a.err, DM_DEVERR_PAGE);
        }
    };
    int last = -1;  // lane i: the last ring position loaded into slot i
    const int page_blocks = 4 * a.Hkv;  // K and V; a tensor-map block coordinate steps over 8 rows
    // K (kv 0) or V (kv 1), or both in pairs, of the tile with these pages into ring position `at`
    auto load = [&](uint32_t at, int id, int h, int kv) {
        const uint32_t si = at % SL;
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ring.empty[si], ((at / SL) & 1u) ^ 1u, a.err, abort_flag)))
            return false;
        if (lane == 0) mbar_arrive_expect_tx(&ring.full[si], kSlot);
        if (lane == static_cast<int>(si)) last = static_cast<int>(at);
        __syncwarp();
        if (lane < kKeyPages) {
            tma_load_page(smem_u32(sm + si * kSlot) + lane * (2 * Tile::kGroup), map, kv,
                          (id < 0 ? a.num_pages : id) * page_blocks + 2 * h, &ring.full[si]);
        }
        return true;
    };
    Group g0, g1, g2;
    fetch_ids(g0);
    fetch_ids(g1);
    fetch_scales(g0);
    uint32_t x = 0;                // tile
    int prev_id = -1, prev_h = 0;  // pages of the tile before, by lane % 8
    while (g0.count > 0 && ok) {
        fetch_ids(g2);
        fetch_scales(g1);
        for (int k = 0; k < g0.count && ok; ++k, ++x) {
            const int from = k * kKeyPages + lane % kKeyPages;
            const int h = __shfl_sync(0xffffffffu, g0.h, from);
            int id = __shfl_sync(0xffffffffu, g0.id, from);
            if (id >= a.num_pages) id = -1;
            const float2 sc = make_float2(__shfl_sync(0xffffffffu, g0.sc.x, from), __shfl_sync(0xffffffffu, g0.sc.y, from));
            if (!(ok = load(ring.k_load(x), id, h, 0))) break;
            if (lane < kKeyPages) ring.meta[x % ring.kMeta][lane] = sc;
            __syncwarp();
            if (lane == 0) mbar_arrive(&ring.meta_full[x % ring.kMeta]);
            if (!PAIR && x > 0) ok = load(ring.v_load(x - 1), prev_id, prev_h, 1);
            prev_id = id;
            prev_h = h;
        }
        g0 = g1;
        g1 = g2;
    }
    if (!PAIR && ok && x > 0) ok = load(ring.v_load(x - 1), prev_id, prev_h, 1);
    // no copy is left in flight, whoever gave up
    if (last >= 0) ring.wait_full(static_cast<uint32_t>(last), a.err, nullptr);
}

}  // namespace dm
