// dm_kv8_attn.cu — attention over the 8-bit paged cache, row-block kernel: any query count,
// head grouping, head dimension and type (C entries dm_kv8_attention,
// dm_kv8_attention_workspace).
//
// Work item: 8 query rows (a row = one query token and one query head) of one request and
// kv head, and one of `nsplit` ranges of its pages.  For one token per request the rows are
// the heads of the group, so a page is read from HBM once for the whole group.
//
// Mathematics (per row, keys in pages of 16): online softmax in base 2 with the running
// maximum m and the sum l; with the page's scales sK, sV = 2^k
//   s = (q . codeK) * sK * sm_scale * log2 e,   p = 2^(s - m),
//   o = (sum p sV codeV) / (sum p).
// The e4m3 codes are exact in fp16, so the products run on the fp16 tensor cores with fp32
// accumulation and no loss on the cache's side.  q is scaled by a power of two per row and
// split into two fp16 terms (22 bits); the 8 rows' high terms fill A rows 0-7 and their low
// terms A rows 8-15 of one m16n8k16 product, whose two halves are summed: the second term
// costs nothing.  The weight p sV enters as 2^12 2^(s + log2 sV - m'), m' the row's running
// maximum of s + log2 sV, so that it stays in fp16's range whatever the page scales are (o has
// its own rescaling, by m'); for fp32 outputs as two fp16 terms, for bf16 outputs as one
// (relative error 2^-12, against the output's own rounding of 2^-9).
//
// Data path: a lane copies with cp.async exactly the bytes that it will feed to the tensor
// cores, into its own slots of a per-warp shared-memory ring, so the ring needs no barrier
// and no bank conflict occurs.  K: lane (g, t) = (lane / 4, lane % 4) takes 16 bytes of
// tokens g and g + 8 per 64-byte chunk (4 K-steps of 4 elements each: which 16 of the head's
// elements form a K-step is free as long as Q uses the same order).  V: tokens 2t, 2t+1,
// 2t+8, 2t+9 and 16 bytes (8 at D = 64) from g * 16; two byte permutes pair the tokens, and
// O^T = V^T P^T takes P straight from the score product's registers as its B operand.
#include <cmath>
#include <cuda_fp8.h>

#include "dm_common.cuh"
#include "dm_kv8.h"

namespace dm {

constexpr int kKaWarps = 4;
constexpr int kKaStages = 3;
constexpr int kKaRows = 8;
constexpr float kKaPBoost = 4096.0f;

template <int D>
struct KaShape {
    static constexpr int kVB = D >= 128 ? 16 : 8;        // V bytes of a lane and token per half
    static constexpr int kHalves = D / (8 * kVB);        // V column groups of 8 lanes * kVB
    static constexpr int kKLoads = 2 * (D / 64);         // 16-byte K loads of a lane and page
    static constexpr int kVLoads = 4 * kHalves;          // kVB-byte V loads of a lane and page
    static constexpr int kStageBytes = 32 * D;           // K and V of one page and kv head
    static constexpr int kTiles = D / 16;                // 16-row tiles of O^T
    static constexpr size_t kSmem = static_cast<size_t>(kKaWarps) * kKaStages * kStageBytes;
    static_assert(kStageBytes * kKaStages >= kKaRows * D * 4, "a warp's ring holds its O block");
};

DM_DEV uint32_t e4m3x2_to_h2(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
    return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
DM_DEV uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
DM_DEV void mma_f16_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
DM_DEV void cp_async8(void* smem_dst, const void* gmem_src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(smem_dst)), "l"(gmem_src) : "memory");
}
template <int N>
DM_DEV void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// 0xff in the bytes of w that hold an e4m3 NaN code
DM_DEV uint32_t e4m3_nan_mask(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

template <typename T, int D>
__global__ void __launch_bounds__(kKaWarps * 32) kv8_attn_rows_kernel(const __grid_constant__ Kv8AttnArgs a) {
    using S = KaShape<D>;
    constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;  // fp16 terms of p
    extern __shared__ __align__(128) uint8_t ka_smem[];
    __shared__ float s_m[kKaWarps][kKaRows], s_l[kKaWarps][kKaRows], s_w[kKaWarps][kKaRows], s_tot[2][kKaRows];
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, tq = lane & 3;

    // work item
    int item = blockIdx.x;
    const int split = item % a.nsplit;
    item /= a.nsplit;
    const int h = item % a.Hkv;
    const int blk = (item / a.Hkv) % a.blocks;
    const int req = item / a.Hkv / a.blocks;
    int row0 = req, m_rows = 1;
    if (a.cu_q) {
        row0 = a.cu_q[req];
        m_rows = a.cu_q[req + 1] - row0;
        if (row0 < 0 || m_rows < 0 || m_rows > a.max_q || row0 > a.rows - m_rows) {
            if (split == 0 && blk == 0 && h == 0 && tid == 0) raise_error(a.err, DM_DEVERR_RANGE);
            return;
        }
    }
    if (blk * kKaRows >= m_rows * a.group) return;
    int len = a.seq_lens[req];
    if (len < 0) {
        if (tid == 0) raise_error(a.err, DM_DEVERR_RANGE);
        len = 0;
    }
    const int full = len;
    if (len > a.width * kKv8Page) {
        if (tid == 0) raise_error(a.err, DM_DEVERR_CAPACITY);
        len = a.width * kKv8Page;
    }
    // this lane's row: keys before `lim` are seen
    const int nrow = min(kKaRows, m_rows * a.group - blk * kKaRows);
    const int fr = blk * kKaRows + min(g, nrow - 1);
    const int tok = fr / a.group, head = h * a.group + fr % a.group;
    const int lim = min(len, max(0, full - m_rows + tok + 1));
    const int tok_first = blk * kKaRows / a.group, tok_last = (blk * kKaRows + nrow - 1) / a.group;
    const int lim_min = min(len, max(0, full - m_rows + tok_first + 1));
    const int lim_max = min(len, max(0, full - m_rows + tok_last + 1));
    const int pages = (lim_max + kKv8Page - 1) / kKv8Page;
    const int per = (pages + a.nsplit - 1) / a.nsplit;
    const int p_begin = min(pages, split * per), p_end = min(pages, p_begin + per);

    uint8_t* ring = ka_smem + static_cast<size_t>(wid) * (kKaStages * S::kStageBytes);
    const int* table = a.table + static_cast<size_t>(req) * a.width;
    const int mine = p_end - p_begin > wid ? (p_end - p_begin - wid + kKaWarps - 1) / kKaWarps : 0;

    // page ids and scales of this warp's next 32 pages, one per lane
    int id_n = -1, id_c = -1;
    float sk_n = 0.0f, sv_n = 0.0f, sk_c = 0.0f, sv_c = 0.0f;
    auto fetch_meta = [&](int base, int& id, float& sk, float& sv) {
        id = -1;
        sk = sv = 0.0f;
        if (base + lane < mine) {
            const int p = table[p_begin + wid + (base + lane) * kKaWarps];
            if (p >= 0 && p < a.num_pages) {
                id = p;
                const float* sc = a.scales + static_cast<size_t>(p) * 2 * a.Hkv + h;
                sk = sc[0];
                sv = sc[a.Hkv];
            } else {
                raise_error(a.err, DM_DEVERR_PAGE);
            }
        }
    };
    auto issue = [&](int it) {  // page `it` of this warp into its ring slot
        const int id = __shfl_sync(0xffffffffu, id_n, it & 31);
        if (id < 0) return;
        uint8_t* st = ring + (it % kKaStages) * S::kStageBytes;
        const uint8_t* k = a.pages + (static_cast<size_t>(id) * 2 * a.Hkv + h) * (kKv8Page * D);
        const uint8_t* v = k + static_cast<size_t>(a.Hkv) * (kKv8Page * D);
#pragma unroll
        for (int i = 0; i < S::kKLoads; ++i)  // i = chunk * 2 + token half
            cp_async16(st + i * 512 + lane * 16, k + ((i & 1) * 8 + g) * D + (i >> 1) * 64 + tq * 16);
        uint8_t* sv = st + kKv8Page * D;
#pragma unroll
        for (int i = 0; i < S::kVLoads; ++i) {  // i = half * 4 + token of the lane
            const int t = 2 * tq + (i & 1) + ((i >> 1) & 1) * 8;
            const uint8_t* src_v = v + t * D + (i >> 2) * (8 * S::kVB) + g * S::kVB;
            if constexpr (S::kVB == 16) cp_async16(sv + i * 512 + lane * 16, src_v);
            else cp_async8(sv + i * 256 + lane * 8, src_v);
        }
    };

    // Q: this lane's row, scaled by a power of two to a largest magnitude in [2^13, 2^14),
    // as fp16 hi + lo
    uint32_t qh[D / 8], ql[D / 8];
    float c_row;
    {
        const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(row0 + tok) * a.q_rs + head * a.q_hs;
        float amax = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(static_cast<float>(q[c * 64 + tq * 16 + e])));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int e = ((__float_as_int(amax) >> 23) & 0xff) - 127 - 13;
        e = max(-100, min(100, e));
        const float mul = __int_as_float((127 - e) << 23);
        c_row = a.scale_log2 * __int_as_float((127 + e) << 23);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = static_cast<float>(q[c * 64 + tq * 16 + 2 * j]) * mul;
                const float y = static_cast<float>(q[c * 64 + tq * 16 + 2 * j + 1]) * mul;
                const uint32_t hi = pack_h2(x, y);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                qh[c * 8 + j] = hi;
                ql[c * 8 + j] = pack_h2(x - f.x, y - f.y);
            }
    }

    float o[S::kTiles][4];
#pragma unroll
    for (int i = 0; i < S::kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m = -INFINITY, mp = -INFINITY, l = 0.0f;  // row g; mp = m' above

    fetch_meta(0, id_n, sk_n, sv_n);
    id_c = id_n, sk_c = sk_n, sv_c = sv_n;
#pragma unroll
    for (int i = 0; i < kKaStages - 1; ++i) {
        if (i < mine) issue(i);
        cp_async_commit();
    }
    for (int it = 0; it < mine; ++it) {
        const int ahead = it + kKaStages - 1;
        if ((it & 31) == 0 && it) id_c = id_n, sk_c = sk_n, sv_c = sv_n;
        if ((ahead & 31) == 0 && ahead < mine) fetch_meta(ahead, id_n, sk_n, sv_n);
        if (ahead < mine) issue(ahead);
        cp_async_commit();
        cp_async_wait<kKaStages - 1>();
        const uint8_t* st = ring + (it % kKaStages) * S::kStageBytes;
        const int key0 = (p_begin + wid + it * kKaWarps) * kKv8Page;
        const bool have = __shfl_sync(0xffffffffu, id_c, it & 31) >= 0;
        const float sk = __shfl_sync(0xffffffffu, sk_c, it & 31), sv = __shfl_sync(0xffffffffu, sv_c, it & 31);

        // scores of tokens key0 + 8 nt + {2 tq, 2 tq + 1} of row g
        float s[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const uint4 k4 = *reinterpret_cast<const uint4*>(st + (c * 2 + nt) * 512 + lane * 16);
                const uint32_t kw[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    mma_f16_m16n8k16(s[nt], qh[c * 8 + 2 * j], ql[c * 8 + 2 * j], qh[c * 8 + 2 * j + 1],
                                     ql[c * 8 + 2 * j + 1], e4m3x2_to_h2(kw[j]), e4m3x2_to_h2(kw[j] >> 16));
            }
        const float f = c_row * sk;
        float p[4] = {(s[0][0] + s[0][2]) * f, (s[0][1] + s[0][3]) * f, (s[1][0] + s[1][2]) * f,
                      (s[1][1] + s[1][3]) * f};
        const bool edge = key0 + kKv8Page > lim_min || !have;
        if (edge) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (!have || key0 + 2 * tq + (j & 1) + (j >> 1) * 8 >= lim) p[j] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m, mx);
        const float mp_new = fmaxf(mp, mx + static_cast<float>(((__float_as_int(sv) >> 23) & 0xff) - 127));
        const float m_use = m_new == -INFINITY ? 0.0f : m_new, mp_use = mp_new == -INFINITY ? 0.0f : mp_new;
        if (__any_sync(0xffffffffu, m_new > m || mp_new > mp)) {
            l *= exp2f(m - m_use);  // 0 while nothing was seen
            const float al = exp2f(mp - mp_use);
            const float a0 = __shfl_sync(0xffffffffu, al, tq * 8), a1 = __shfl_sync(0xffffffffu, al, tq * 8 + 4);
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) {
                o[i][0] *= a0, o[i][1] *= a1, o[i][2] *= a0, o[i][3] *= a1;
            }
            m = m_new;
            mp = mp_new;
        }
        const float fv = sv * exp2f(m_use - mp_use) * kKaPBoost;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] = exp2f(p[j] - m_use);
            l += p[j];
        }
        uint32_t ph[2], pl[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float x = p[2 * j] * fv, y = p[2 * j + 1] * fv;
            ph[j] = pack_h2(x, y);
            if constexpr (kTerms == 2) {
                const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&ph[j]));
                pl[j] = pack_h2(x - hf.x, y - hf.y);
            }
        }
        // V: zeros behind the last key; on pages that not every row sees, a NaN code must reach
        // only the rows that see it, so it becomes 0 and makes those rows' sums NaN
        uint32_t nan_tok = 0;
        const uint8_t* stv = st + kKv8Page * D;
#pragma unroll
        for (int hf = 0; hf < S::kHalves; ++hf) {
            uint32_t w[4][S::kVB / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (S::kVB == 16) {
                    const uint4 u = *reinterpret_cast<const uint4*>(stv + (hf * 4 + i) * 512 + lane * 16);
                    w[i][0] = u.x, w[i][1] = u.y, w[i][2] = u.z, w[i][3] = u.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(stv + (hf * 4 + i) * 256 + lane * 8);
                    w[i][0] = u.x, w[i][1] = u.y;
                }
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool dead = !have || key0 + 2 * tq + (i & 1) + (i >> 1) * 8 >= lim_max;
#pragma unroll
                    for (int j = 0; j < S::kVB / 4; ++j) {
                        const uint32_t bad = dead ? 0xffffffffu : e4m3_nan_mask(w[i][j]);
                        w[i][j] &= ~bad;
                        if (!dead && bad) nan_tok |= 1u << i;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < S::kVB / 4; ++j) {
                const uint32_t x0 = __byte_perm(w[0][j], w[1][j], 0x5140), x1 = __byte_perm(w[0][j], w[1][j], 0x7362);
                const uint32_t y0 = __byte_perm(w[2][j], w[3][j], 0x5140), y1 = __byte_perm(w[2][j], w[3][j], 0x7362);
                const int ti = hf * (S::kVB / 2) + 2 * j;
                const uint32_t a00 = e4m3x2_to_h2(x0), a01 = e4m3x2_to_h2(x0 >> 16), a02 = e4m3x2_to_h2(y0),
                               a03 = e4m3x2_to_h2(y0 >> 16);
                const uint32_t a10 = e4m3x2_to_h2(x1), a11 = e4m3x2_to_h2(x1 >> 16), a12 = e4m3x2_to_h2(y1),
                               a13 = e4m3x2_to_h2(y1 >> 16);
                mma_f16_m16n8k16(o[ti], a00, a01, a02, a03, ph[0], ph[1]);
                mma_f16_m16n8k16(o[ti + 1], a10, a11, a12, a13, ph[0], ph[1]);
                if constexpr (kTerms == 2) {
                    mma_f16_m16n8k16(o[ti], a00, a01, a02, a03, pl[0], pl[1]);
                    mma_f16_m16n8k16(o[ti + 1], a10, a11, a12, a13, pl[0], pl[1]);
                }
            }
        }
        if (edge) {
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) nan_tok |= __shfl_xor_sync(0xffffffffu, nan_tok, x);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if ((nan_tok >> i & 1) && key0 + 2 * tq + (i & 1) + (i >> 1) * 8 < lim)
                    l = __int_as_float(0x7fc00000);
        }
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);

    // join the warps: O to shared memory as [row][D] in true units
    cp_async_wait_all();
    if (tq == 0) {
        s_m[wid][g] = m;
        s_l[wid][g] = l;
    }
    float* ow = reinterpret_cast<float*>(ring);
    {
        const float u = m == -INFINITY ? 0.0f : exp2f(mp - m) * (1.0f / kKaPBoost);
        const float u0 = __shfl_sync(0xffffffffu, u, tq * 8), u1 = __shfl_sync(0xffffffffu, u, tq * 8 + 4);
        // lane (g, tq) holds heads 2 tq, 2 tq + 1 and, per tile ti, elements d, d + 1
#pragma unroll
        for (int ti = 0; ti < S::kTiles; ++ti) {
            const int d = (ti / (S::kVB / 2)) * (8 * S::kVB) + g * S::kVB + 2 * (ti % (S::kVB / 2));
            *reinterpret_cast<float2*>(ow + (2 * tq) * D + d) = make_float2(o[ti][0] * u0, o[ti][2] * u0);
            *reinterpret_cast<float2*>(ow + (2 * tq + 1) * D + d) = make_float2(o[ti][1] * u1, o[ti][3] * u1);
        }
    }
    __syncthreads();
    if (tid < kKaRows) {
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) mm = fmaxf(mm, s_m[w][tid]);
        const float mu = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) {
            const float x = exp2f(s_m[w][tid] - mu);
            s_w[w][tid] = x;
            // a NaN sum stays NaN; a warp without keys has l = 0
            ll += s_l[w][tid] * x;
        }
        s_tot[0][tid] = mm;
        s_tot[1][tid] = ll;
    }
    __syncthreads();
    constexpr int kRing = kKaStages * S::kStageBytes / 4;  // floats between the warps' blocks
    const float* all = reinterpret_cast<const float*>(ka_smem);
    auto joined = [&](int r, int d) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) x += all[w * kRing + r * D + d] * s_w[w][r];
        return x;
    };
    auto put = [&](int r, int d, float x, float mm, float ll) {
        const int f2 = blk * kKaRows + r;
        const int64_t row = row0 + f2 / a.group;
        const int hd = h * a.group + f2 % a.group;
        static_cast<T*>(a.out)[row * a.o_rs + hd * a.o_hs + d] = static_cast<T>(mm == -INFINITY ? 0.0f : x / ll);
        if (d == 0 && a.lse)
            a.lse[row * a.Hq + hd] = mm == -INFINITY ? -INFINITY : mm * 0.6931471805599453f + logf(ll);
    };
    if (a.nsplit == 1) {
        for (int i = tid; i < nrow * D; i += blockDim.x) {
            const int r = i / D, d = i % D;
            put(r, d, joined(r, d), s_tot[0][r], s_tot[1][r]);
        }
        return;
    }
    // partial of this split; the last split of the item to arrive joins them in split order
    constexpr int kSlot = kKaRows * (D + 2);
    float* part = a.part + (static_cast<size_t>(item) * a.nsplit + split) * kSlot;
    for (int i = tid; i < nrow * D; i += blockDim.x) part[i] = joined(i / D, i % D);
    if (tid < nrow) {
        part[kKaRows * D + tid] = s_tot[0][tid];
        part[kKaRows * D + kKaRows + tid] = s_tot[1][tid];
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        const unsigned got = atomicAdd(a.counters + item, 1u);
        s_last = got == static_cast<unsigned>(a.nsplit) - 1;
        if (s_last) a.counters[item] = 0;
        __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    const float* base = a.part + static_cast<size_t>(item) * a.nsplit * kSlot;
    for (int i = tid; i < nrow * D; i += blockDim.x) {
        const int r = i / D, d = i % D;
        float mm = -INFINITY;
        for (int sp = 0; sp < a.nsplit; ++sp) mm = fmaxf(mm, __ldcg(base + sp * kSlot + kKaRows * D + r));
        const float mu = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f, x = 0.0f;
        for (int sp = 0; sp < a.nsplit; ++sp) {
            const float* b = base + sp * kSlot;
            const float wgt = exp2f(__ldcg(b + kKaRows * D + r) - mu);
            ll += __ldcg(b + kKaRows * D + kKaRows + r) * wgt;
            x += __ldcg(b + i) * wgt;
        }
        put(r, d, x, mm, ll);
    }
}

// Splits: enough CTAs for two waves of two per SM, no split without a page of its own for
// every warp, and at most kMaxSlots partials (the workspace).
constexpr int kKaMaxSlots = 2048;

template <typename T, int D>
static cudaError_t launch_rows(const Kv8AttnArgs& a, cudaStream_t s) {
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
        e = cudaFuncSetAttribute(kv8_attn_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(KaShape<D>::kSmem));
        if (e == cudaSuccess && dev < 64) ready[dev] = true;
    }
    if (e != cudaSuccess) return e;
    const unsigned grid = static_cast<unsigned>(a.n) * a.blocks * a.Hkv * a.nsplit;
    kv8_attn_rows_kernel<T, D><<<grid, kKaWarps * 32, KaShape<D>::kSmem, s>>>(a);
    return cudaGetLastError();
}

static size_t workspace_bytes(int D) {
    return static_cast<size_t>(kKaMaxSlots) * kKaRows * (D + 2) * sizeof(float) + kKaMaxSlots * sizeof(unsigned);
}

}  // namespace dm

using namespace dm;

extern "C" int32_t dm_kv8_attention_workspace(const dm_kv8_cache* c, uint64_t* bytes, char* eb, uint64_t es) {
    const char* st = "kv8_attention";
    if (eb && es > 0) eb[0] = '\0';
    if (int rc = kv8_check_cache(c, st, eb, es)) return rc;
    if (!bytes) return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    *bytes = workspace_bytes(c->head_dim);
    return DM_OK;
}

extern "C" int32_t dm_kv8_attention(const dm_kv8_cache* c, const dm_kv8_attn_args* p, void* stream, char* eb,
                                    uint64_t es) {
    const char* st = "kv8_attention";
    if (eb && es > 0) eb[0] = '\0';
    if (int rc = kv8_check_cache(c, st, eb, es)) return rc;
    if (!p) return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null arguments");
    if (p->dtype != DM_DTYPE_BF16 && p->dtype != DM_DTYPE_F32)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "dtype is bf16 or fp32");
    if (p->n < 0 || p->rows < 0 || p->reserved != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "negative n or rows, or reserved not 0");
    if (p->num_q_heads < 1 || p->num_q_heads % c->num_kv_heads != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", st, "num_q_heads %d is no multiple of %d kv heads",
                       p->num_q_heads, c->num_kv_heads);
    if (!std::isfinite(p->sm_scale))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "sm_scale is not finite");
    if (p->table_width < 1 || p->table_width >= (1 << 27))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "table_width %d", p->table_width);
    if (p->max_q_len < 1 || (!p->cu_q && (p->max_q_len != 1 || p->rows < p->n)))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st,
                       "need max_q_len >= 1; without cu_q max_q_len is 1 and rows >= n");
    if (p->n == 0 || p->rows == 0) return DM_OK;
    if (!p->q || !p->out || !p->block_table || !p->seq_lens || !p->workspace)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    if (reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0 || p->workspace_bytes < workspace_bytes(c->head_dim))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st,
                       "the workspace needs %llu bytes at a multiple of 256 (given %llu)",
                       static_cast<unsigned long long>(workspace_bytes(c->head_dim)),
                       static_cast<unsigned long long>(p->workspace_bytes));
    Kv8AttnArgs a{};
    a.group = p->num_q_heads / c->num_kv_heads;
    const int64_t max_q = p->max_q_len < p->rows ? p->max_q_len : p->rows;
    const int64_t blocks = (max_q * a.group + kKaRows - 1) / kKaRows;
    const int64_t items = blocks * p->n * c->num_kv_heads;
    if (items >= (1LL << 31))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "too many query rows for one call");
    Kv8Device g;
    if (int rc = g.enter(c->pages, st, eb, es)) return rc;
    a.pages = c->pages;
    a.scales = c->scales;
    a.q = p->q, a.q_rs = p->q_row_stride, a.q_hs = p->q_head_stride;
    a.out = p->out, a.o_rs = p->out_row_stride, a.o_hs = p->out_head_stride;
    a.lse = p->lse;
    a.table = p->block_table;
    a.seq_lens = p->seq_lens;
    a.cu_q = p->cu_q;
    a.err = p->err_dev;
    a.scale_log2 = p->sm_scale * 1.4426950408889634f;
    a.n = p->n;
    a.rows = p->rows;
    a.Hq = p->num_q_heads;
    a.Hkv = c->num_kv_heads;
    a.num_pages = c->num_pages;
    a.width = p->table_width;
    a.max_q = static_cast<int>(p->max_q_len);
    a.blocks = static_cast<int>(blocks);
    int64_t split = 4LL * g.num_sms / items;
    const int64_t most = (p->table_width + kKaWarps - 1) / kKaWarps;
    if (split > most) split = most;
    if (split < 1) split = 1;
    if (split > 1 && items * split > kKaMaxSlots) split = kKaMaxSlots / items;
    a.nsplit = static_cast<int>(split < 1 ? 1 : split);
    a.counters = static_cast<unsigned*>(p->workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + kKaMaxSlots * sizeof(unsigned));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    const bool f32 = p->dtype == DM_DTYPE_F32;
    switch (c->head_dim) {
        case 64: e = f32 ? launch_rows<float, 64>(a, s) : launch_rows<__nv_bfloat16, 64>(a, s); break;
        case 128: e = f32 ? launch_rows<float, 128>(a, s) : launch_rows<__nv_bfloat16, 128>(a, s); break;
        default: e = f32 ? launch_rows<float, 256>(a, s) : launch_rows<__nv_bfloat16, 256>(a, s); break;
    }
    if (e != cudaSuccess)
        return kv8_err(eb, es, e == cudaErrorInvalidValue ? DM_ERR_INVALID_ARG : DM_ERR_CUDA, "CUDA_ERROR", st,
                       "launch: %s", cudaGetErrorString(e));
    return DM_OK;
}
