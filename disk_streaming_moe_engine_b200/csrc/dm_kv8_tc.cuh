// dm_kv8_tc.cuh — tcgen05 kind::f8f6f4 (e4m3 x e4m3 -> fp32) and TMA helpers of the 8-bit
// cache attention kernels.
//
// Operand tiles in shared memory: blocks of 8 rows by CW bytes (CW = 128 with the 128-byte
// swizzle, or 64 with the 64-byte swizzle at head_dim 64), the 16-byte units of a row permuted by
// the row.  The same cache bytes serve two roles: K as a K-major operand (rows = M, the head's
// elements = K) and V as an M- or N-major operand (rows = K, the head's elements = M or N).
#pragma once
#include <cuda.h>
#include <cuda_fp8.h>

#include "dm_kv8.h"
#include "dm_tc.cuh"

namespace dm {

constexpr uint64_t kDescVersion = 1ull << 46;

// K-major operand of CW-byte rows: 8-row blocks `group` bytes apart (stride byte offset); one
// K = 32 step of the tile advances the start address by 32 bytes.
template <int CW>
DM_DEV uint64_t f8_desc_k(uint32_t addr, uint32_t group) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(group / 16) << 32) |
           kDescVersion | (static_cast<uint64_t>(CW == 128 ? 2 : 4) << 61);
}
// M- or N-major operand: 8-token blocks `group` bytes apart (stride byte offset), the next CW
// elements of M or N `chunk` bytes on (leading byte offset; 0 repeats the first CW elements).
template <int CW>
DM_DEV uint64_t f8_desc_m(uint32_t addr, uint32_t chunk, uint32_t group) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(chunk / 16) << 16) |
           (static_cast<uint64_t>(group / 16) << 32) | kDescVersion | (static_cast<uint64_t>(CW == 128 ? 2 : 4) << 61);
}
// N-major operand without swizzle: per 16 N columns a block of 16-byte rows, one per K;
// 8-row groups 128 bytes apart (leading byte offset), blocks `block` bytes apart (stride).
DM_DEV uint64_t f8_desc_n16(uint32_t addr, uint32_t block) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 / 16) << 16) |
           (static_cast<uint64_t>(block / 16) << 32) | kDescVersion;
}

// Instruction descriptor: fp32 accumulator, e4m3 operands; bit 15 / 16: A / B with M / N as
// the contiguous dimension.
DM_DEV uint32_t f8_idesc(int M, int N, bool a_m_major, bool b_n_major) {
    return (1u << 4) | (a_m_major ? 1u << 15 : 0u) | (b_n_major ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

DM_DEV void f8_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

// The same with A in tensor memory: row m in lane m, four consecutive K elements per 32-bit
// column, 8 columns per K = 32 step.
DM_DEV void f8_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

// A page's box: block coordinate `block`, from K (kv 0) or V (kv 1) on.
DM_DEV void tma_load_page(uint32_t smem_dst, const CUtensorMap* map, int kv, int block, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, "
        "%4}], [%5];" ::"r"(smem_dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(kv), "r"(block), "r"(smem_u32(bar))
        : "memory");
}

// Byte of 16-byte unit u of token row r in a tile of CW-byte rows.
template <int CW>
DM_DEV uint32_t f8_unit(int r, int u) {
    const int x = CW == 128 ? (u ^ (r & 7)) : (u ^ ((r >> 1) & 3));
    return static_cast<uint32_t>(r * CW + x * 16);
}

// Codes of two fp16 values (a in the low byte), and 16 times what they leave (exact).
DM_DEV uint32_t e4m3_take2(__half2& h) {
    const uint32_t c = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(h), __NV_SATFINITE, __NV_E4M3);
    const __half2 back(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c), __NV_E4M3));
    h = __hmul2(__hsub2(h, back), __float2half2_rn(16.0f));
    return c;
}
// e4m3 terms of two values of magnitude up to 448, term i scaled by 2^4i.  Two terms hold 8 bits of
// the value as fp16, three its 11; with five the first three take its 11 bits and the other two 8 bits
// of the rest, 2^12 times of which is an fp16 value again: 2^-20 of the value, or 2^-26.
template <int TERMS>
DM_DEV void e4m3_split2(float a, float b, uint32_t (&t)[TERMS]) {
    static_assert(TERMS == 2 || TERMS == 3 || TERMS == 5, "terms");
    __half2 h = __floats2half2_rn(a, b);
    __half2 rest = h;
    if constexpr (TERMS == 5) {
        const float2 f = __half22float2(h);
        rest = __floats2half2_rn((a - f.x) * 4096.0f, (b - f.y) * 4096.0f);
    }
    t[0] = e4m3_take2(h);
    t[1] = e4m3_take2(h);
    if constexpr (TERMS > 2) t[2] = e4m3_take2(h);
    if constexpr (TERMS == 5) {
        rest = __hadd2(rest, h);  // what small values still have left, at the same scale
        t[3] = e4m3_take2(rest);
        t[4] = e4m3_take2(rest);
    }
}
// 0xff in byte i where value i has its sign bit set
DM_DEV uint32_t sign_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    uint32_t lo, hi;
    asm("prmt.b32 %0, %1, %2, 0xFB;" : "=r"(lo) : "r"(a), "r"(b));  // 8 + i: the sign of byte i
    asm("prmt.b32 %0, %1, %2, 0xFB;" : "=r"(hi) : "r"(c), "r"(d));
    return __byte_perm(lo, hi, 0x5410);
}
// 0xff in the bytes of w that hold a NaN code
DM_DEV uint32_t e4m3_nan_mask(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// e4m3 terms of two values: the nearest codes, and those of what they leave (as they are, no
// scaling), through fp16 (11 bits, twice what the two terms hold)
DM_DEV void e4m3_terms2(float a, float b, uint32_t& t0, uint32_t& t1) {
    const __half2 h = __floats2half2_rn(a, b);
    t0 = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(h), __NV_SATFINITE, __NV_E4M3);
    const __half2 back(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(t0), __NV_E4M3));
    t1 = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(__hsub2(h, back)), __NV_SATFINITE, __NV_E4M3);
}

// Three e5m2 terms of four values in [0, 2^15], all of one scale, a byte each.  An e5m2 code is the
// upper byte of an fp16 value: three of its bits at a time stay with their exponent, what they leave
// is exact, and the last term is rounded (conversion instructions took 40 % longer).
DM_DEV void e5m2_terms3(float a, float b, float c, float d, uint32_t (&t)[3]) {
    uint32_t x[2], top[2];
    const __half2 h0 = __floats2half2_rn(a, b), h1 = __floats2half2_rn(c, d);
    x[0] = *reinterpret_cast<const uint32_t*>(&h0);
    x[1] = *reinterpret_cast<const uint32_t*>(&h1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            top[j] = x[j] & 0xff00ff00u;
            const __half2 rest = __hsub2(*reinterpret_cast<const __half2*>(&x[j]), *reinterpret_cast<const __half2*>(&top[j]));
            x[j] = *reinterpret_cast<const uint32_t*>(&rest);
        }
        t[i] = __byte_perm(top[0], top[1], 0x7531);
    }
    t[2] = __byte_perm(x[0] + 0x00800080u, x[1] + 0x00800080u, 0x7531);
}

// 32 bytes of one thread (32-byte aligned): whole sectors where every lane has a row of its own
DM_DEV void ldg_v8(uint32_t* v, const void* p) {
    asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(p));
}
DM_DEV void stg_v8(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// larger of each half (bf16 pairs); NaN wins
DM_DEV uint32_t bf16x2_max_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// 2^x of the special function unit (relative error 2^-22; results below 2^-126 become 0)
DM_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Counts an arrival: what the CTA wrote before its last barrier is visible to whoever sees the
// count, and what the others wrote before theirs to this CTA after its next barrier.
DM_DEV unsigned atom_add_acq_rel(unsigned* p, unsigned v) {
    unsigned old;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
    return old;
}

// Barrier over `count` threads that also ORs a predicate.
DM_DEV bool named_bar_or(int id, int count, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %3, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(count), "r"(v ? 1u : 0u)
        : "memory");
    return r != 0;
}

// Tensor map of the cache: (CW bytes, 8 rows, chunk of the head, K | V, 8-row block of the cache
// counted over page, kv head and half page as if there were no K | V), boxes of a page's two
// blocks with all chunks and K alone, V alone or, in pairs, both.  A block behind the last page
// reads zeros.  One copy per page (8 KB in pairs at head_dim 256) instead of one per 2 KB.
bool kv8_encode_map(const dm_kv8_cache* c, bool pair, CUtensorMap* map);

}  // namespace dm
