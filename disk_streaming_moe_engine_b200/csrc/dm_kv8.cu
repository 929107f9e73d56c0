// dm_kv8.cu — slot planning, rotary positions and the quantising append of the 8-bit paged
// KV cache (C entries dm_kv8_plan, dm_rope, dm_kv8_append, dm_kv8_status).
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <cuda_fp8.h>

#include "dm_common.cuh"
#include "dm_kv8.h"

namespace dm {

int kv8_err(char* buf, uint64_t size, int code, const char* type, const char* stage, const char* fmt, ...) {
    if (buf && size > 0) {
        char detail[384];
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(detail, sizeof detail, fmt, ap);
        va_end(ap);
        for (char* p = detail; *p; ++p)
            if (*p == '"' || *p == '\\') *p = '\'';
        snprintf(buf, size, "{\"error_type\":\"%s\",\"detail\":\"%s\",\"stage\":\"%s\",\"layer\":-1}", type, detail,
                 stage);
    }
    return code;
}

int Kv8Device::enter(const void* p, const char* stage, char* eb, uint64_t es) {
    cudaPointerAttributes at{};
    cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return kv8_err(eb, es, DM_ERR_CUDA, "CUDA_ERROR", stage, "no device: %s", cudaGetErrorString(e));
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", stage, "a buffer is not device memory");
    int cur = -1;
    e = cudaGetDevice(&cur);
    if (e == cudaSuccess && cur != at.device) {
        e = cudaSetDevice(at.device);
        if (e == cudaSuccess) prev = cur;
    }
    dev = at.device;
    static std::atomic<int> sms[64];  // per device, once known
    const bool known = dev < 64;
    num_sms = known ? sms[dev].load(std::memory_order_relaxed) : 0;
    if (e == cudaSuccess && num_sms == 0) {
        e = cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess && known) sms[dev].store(num_sms, std::memory_order_relaxed);
    }
    if (e != cudaSuccess)
        return kv8_err(eb, es, DM_ERR_CUDA, "CUDA_ERROR", stage, "%s", cudaGetErrorString(e));
    return DM_OK;
}

Kv8Device::~Kv8Device() {
    if (prev >= 0) cudaSetDevice(prev);
}

static __device__ uint32_t g_kv8_err;

uint32_t* kv8_error_word(uint32_t* callers, int dev) {
    if (callers) return callers;
    static std::atomic<void*> at[64];  // per device, once known
    void* p = dev < 64 ? at[dev].load(std::memory_order_relaxed) : nullptr;
    if (!p) {
        if (cudaGetSymbolAddress(&p, g_kv8_err) != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        if (dev < 64) at[dev].store(p, std::memory_order_relaxed);
    }
    return static_cast<uint32_t*>(p);
}

int kv8_check_cache(const dm_kv8_cache* c, const char* stage, char* eb, uint64_t es) {
    if (!c || !c->pages || !c->scales)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", stage, "null cache");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", stage, "head_dim %d: 64, 128 or 256", c->head_dim);
    if (c->num_kv_heads < 1 || c->num_kv_heads > 1024 || c->num_pages < 1 || c->num_pages > (1 << 27) - 1 ||
        (static_cast<int64_t>(c->num_pages) + 1) * 4 * c->num_kv_heads > 0x7fffffffLL || c->reserved != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", stage,
                       "need 1 <= num_kv_heads <= 1024, 1 <= num_pages < 2^27, 4 num_kv_heads (num_pages + 1) < 2^31, "
                       "reserved 0");
    if (reinterpret_cast<uintptr_t>(c->pages) % 16 != 0 || reinterpret_cast<uintptr_t>(c->scales) % 4 != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", stage, "pages must be 16-byte aligned");
    return DM_OK;
}

static int launch_status(cudaError_t e, const char* stage, char* eb, uint64_t es) {
    if (e == cudaSuccess) return DM_OK;
    return kv8_err(eb, es, e == cudaErrorInvalidValue ? DM_ERR_INVALID_ARG : DM_ERR_CUDA, "CUDA_ERROR", stage,
                   "launch: %s", cudaGetErrorString(e));
}

// ---- slot planning ---------------------------------------------------------------------
// One pass over the request lengths gives three prefix sums (new tokens, new pages, released
// pages); every CTA computes them for itself from the 8 n bytes of lengths (n <= 8192, a few
// hundred ns) so that the token arrays are filled by many CTAs in the same launch, without a
// second kernel.  Reads and writes of the step never meet: new table entries lie behind the
// ones that are read, released pages land at or above the count that the pops read below.
// Only in-place lengths or an in-place count have to wait until every CTA has read them; the
// last CTA to arrive writes those.  What bounds it is that chain (lengths, three scans, a binary
// search per token, a dependent table or stack read, the store), not its bytes: 64 requests with a
// token each 3.4 us, 512 requests with up to 1000 new tokens each 7.5 us in a graph; a
// call from Python costs 17 us of host time, the caller's torch allocation among it.
struct Kv8PlanArgs {
    const int* ctx;
    const int* add;
    int* table;
    int* free_pages;
    const int* state;
    int* state_out;
    int* seq_lens;
    int* cu_new;
    int* slots;
    int* positions;
    int* requests;
    uint32_t* err;
    int n, width, cap, max_tokens, in_place;
};

constexpr int kPlanItems = DM_KV8_MAX_REQUESTS / 1024;  // requests per thread at most

// largest i with pre[i] <= x, pre ascending with pre[0] = 0 (runs of equal values: the last)
DM_DEV int plan_find(const unsigned* pre, int n, unsigned x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(1024) kv8_plan_kernel(const __grid_constant__ Kv8PlanArgs a) {
    extern __shared__ unsigned plan_smem[];
    const int n = a.n, tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, wid = tid >> 5;
    unsigned* p_tok = plan_smem;          // [n + 1] exclusive prefix sums
    unsigned* p_add = p_tok + n + 1;      // [n + 1]
    unsigned* p_back = p_add + n + 1;     // [n + 1]
    __shared__ unsigned w_sum[3][32];
    __shared__ unsigned s_last;

    const int per = (n + nt - 1) / nt;
    unsigned tok[kPlanItems], add[kPlanItems], back[kPlanItems];
    unsigned st = 0, sa = 0, sb = 0;
    int bad = 0, bad_range = 0;
    const int count = a.state[0];
#pragma unroll
    for (int j = 0; j < kPlanItems; ++j) {
        tok[j] = add[j] = back[j] = 0;
        const int i = tid * per + j;
        if (j >= per || i >= n) continue;
        const int c = a.ctx[i], w = a.add[i];
        if (c < 0 || w < -1) {
            bad_range = 1;
            continue;
        }
        const long long end = static_cast<long long>(c) + (w > 0 ? w : 0);
        const long long have = (static_cast<long long>(c) + kKv8Page - 1) / kKv8Page;
        const long long need = (end + kKv8Page - 1) / kKv8Page;
        if (need > a.width || end > 0x7fffffffLL) {
            bad = 1;
            continue;
        }
        tok[j] = w > 0 ? w : 0;
        add[j] = w < 0 ? 0u : static_cast<unsigned>(need - have);
        back[j] = w < 0 ? static_cast<unsigned>(have) : 0u;
        st += tok[j];
        sa += add[j];
        sb += back[j];
    }
    // block-wide exclusive scan of the three sums (n * width <= 2^27 keeps them in 32 bits)
    unsigned xt = st, xa = sa, xb = sb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned yt = __shfl_up_sync(0xffffffffu, xt, o), ya = __shfl_up_sync(0xffffffffu, xa, o),
                       yb = __shfl_up_sync(0xffffffffu, xb, o);
        if (lane >= o) {
            xt += yt;
            xa += ya;
            xb += yb;
        }
    }
    if (lane == 31) {
        w_sum[0][wid] = xt;
        w_sum[1][wid] = xa;
        w_sum[2][wid] = xb;
    }
    bad_range = __syncthreads_or(bad_range);
    unsigned bt = 0, ba = 0, bb = 0, total = 0, need_pages = 0, released = 0;
    {
        const int nw = nt >> 5;
        const unsigned vt = lane < nw ? w_sum[0][lane] : 0u, va = lane < nw ? w_sum[1][lane] : 0u,
                       vb = lane < nw ? w_sum[2][lane] : 0u;
        bt = __reduce_add_sync(0xffffffffu, lane < wid ? vt : 0u);
        ba = __reduce_add_sync(0xffffffffu, lane < wid ? va : 0u);
        bb = __reduce_add_sync(0xffffffffu, lane < wid ? vb : 0u);
        total = __reduce_add_sync(0xffffffffu, vt);
        need_pages = __reduce_add_sync(0xffffffffu, va);
        released = __reduce_add_sync(0xffffffffu, vb);
    }
    bt += xt - st;
    ba += xa - sa;
    bb += xb - sb;
#pragma unroll
    for (int j = 0; j < kPlanItems; ++j) {
        const int i = tid * per + j;
        if (j >= per || i >= n) continue;
        p_tok[i] = bt;
        p_add[i] = ba;
        p_back[i] = bb;
        bt += tok[j];
        ba += add[j];
        bb += back[j];
    }
    if (tid == 0) {
        p_tok[n] = total;
        p_add[n] = need_pages;
        p_back[n] = released;
    }
    const long long avail = static_cast<long long>(count) + released;
    if (count < 0 || avail > a.cap || need_pages > avail || total > static_cast<unsigned>(a.max_tokens)) bad = 1;
    bad = __syncthreads_or(bad);
    const bool refused = bad || bad_range;
    const int top = static_cast<int>(avail);

    // a page of the stack below `top`: free, or the x-th released one
    auto stack_at = [&](int idx) -> int {
        if (idx < count) return a.free_pages[idx];
        const unsigned x = static_cast<unsigned>(idx - count);
        const int r = plan_find(p_back, n, x);
        return a.table[static_cast<size_t>(r) * a.width + (x - p_back[r])];
    };
    const int gsz = gridDim.x * nt, g0 = blockIdx.x * nt + tid;
    for (int t = g0; t < a.max_tokens; t += gsz) {
        int slot = -1, pos = -1, req = -1;
        if (!refused && static_cast<unsigned>(t) < total) {
            req = plan_find(p_tok, n, t);
            const int c = a.ctx[req];
            pos = c + (t - static_cast<int>(p_tok[req]));
            const int pg = pos / kKv8Page, have = (c + kKv8Page - 1) / kKv8Page;
            const int page = pg < have ? a.table[static_cast<size_t>(req) * a.width + pg]
                                       : stack_at(top - 1 - (static_cast<int>(p_add[req]) + pg - have));
            if (page >= 0 && page < (1 << 27)) slot = page * kKv8Page + pos % kKv8Page;
            else raise_error(a.err, DM_DEVERR_PAGE);
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
        a.requests[t] = req;
    }
    if (!refused) {
        for (int j = g0; j < static_cast<int>(need_pages); j += gsz) {
            const int r = plan_find(p_add, n, j);
            const int have = (a.ctx[r] + kKv8Page - 1) / kKv8Page;
            a.table[static_cast<size_t>(r) * a.width + have + (j - static_cast<int>(p_add[r]))] = stack_at(top - 1 - j);
        }
        for (int x = g0; x < static_cast<int>(released) - static_cast<int>(need_pages); x += gsz)
            a.free_pages[count + x] = stack_at(count + x);
    }
    // lengths, prefix sums and the count: by CTA 0, or by the last CTA when they are in place
    if (a.in_place && gridDim.x > 1) {
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            s_last = atomicAdd(reinterpret_cast<unsigned*>(a.state_out + 1), 1u) == gridDim.x - 1;
            __threadfence();
        }
        __syncthreads();
        if (!s_last) return;
    } else {
        if (blockIdx.x != 0) return;
        __syncthreads();
    }
    for (int i = tid; i <= n; i += nt) {
        a.cu_new[i] = refused ? 0 : static_cast<int>(p_tok[i]);
        if (i < n) {
            const int c = a.ctx[i];
            a.seq_lens[i] = refused ? c : a.add[i] < 0 ? 0 : c + static_cast<int>(p_tok[i + 1] - p_tok[i]);
        }
    }
    if (tid == 0) {
        a.state_out[0] = refused ? count : top - static_cast<int>(need_pages);
        a.state_out[1] = 0;
        if (bad_range) raise_error(a.err, DM_DEVERR_RANGE);
        if (bad) raise_error(a.err, DM_DEVERR_CAPACITY);
    }
}

// ---- rotary positions ---------------------------------------------------------------------
// The angle pos * f is reduced to [-pi, pi] in 64 bits (at position 10^6 an fp32 angle has
// lost 4 decimal digits); the reduced angle goes to fp32 as hi + lo, sin and cos of hi by
// sincosf and the lo part to first order, so both are within an fp32 rounding or two.  The
// angles of a CTA's tokens are computed once and used by every head.  Bound by the bytes, each
// read and written once: 32771 tokens of 32 + 8 heads of 128, all of a head turned, take 116 us or
// 5.77 TB/s (0.89 of the measured copy bandwidth); 64 tokens of 16 + 2 heads 3.65 us, the chain of
// position, angle, barrier, store.  Sixteen tokens per CTA, four tokens' loads in flight, loads and
// stores marked streaming and smaller register budgets gave nothing or cost 1 to 4 us.
struct RopeArgs {
    dm_rope_plan plan;
    const void* x[2];
    void* y[2];
    int64_t x_rs[2], x_hs[2], y_rs[2], y_hs[2];
    int heads[2];
    const int* positions;
    int n, tok, inplace[2];
};

constexpr int kRopeTok = 8;    // tokens of a CTA at most
constexpr int kRopeBatch = 2;  // tokens whose loads a thread has in flight

// 16 bytes (VEC elements) or one element (VEC = 1) as loaded, and as floats
template <typename T, int VEC>
struct RopeVec {
    uint4 u;
    DM_DEV void load(const T* p) {
        if constexpr (VEC == 1) u.x = __float_as_uint(static_cast<float>(p[0]));
        else u = *reinterpret_cast<const uint4*>(p);
    }
    DM_DEV void unpack(float (&v)[VEC]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < (VEC == 1 ? 1 : 4); ++i) {
            if constexpr (VEC != 8) {
                v[i] = __uint_as_float(w[i]);
            } else {
                v[2 * i] = bf16lo(w[i]);
                v[2 * i + 1] = bf16hi(w[i]);
            }
        }
    }
    DM_DEV void store(T* p) const {
        if constexpr (VEC == 1) p[0] = static_cast<T>(__uint_as_float(u.x));
        else *reinterpret_cast<uint4*>(p) = u;
    }
    DM_DEV void pack(const float (&v)[VEC]) {
        if constexpr (VEC == 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            u = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            u.x = __float_as_uint(v[0]);
            if constexpr (VEC == 4)
                u.y = __float_as_uint(v[1]), u.z = __float_as_uint(v[2]), u.w = __float_as_uint(v[3]);
        }
    }
};

// VEC elements per access (16 bytes, or 1 when a pointer or stride is not a multiple of 16
// bytes).  A unit of a head is VEC pairs (half layout: two accesses; interleaved: two
// neighbouring ones, or one pair when VEC = 1) or VEC elements that pass through; a thread
// keeps its unit over the CTA's tokens, and its first batch of loads is in flight while the
// CTA computes the angles.
template <typename T, int VEC>
__global__ void __launch_bounds__(512) rope_kernel(const __grid_constant__ RopeArgs a) {
    __shared__ float2 cs[kRopeTok][128];  // pair unit * VEC + k at k * units + unit: no bank conflicts
    __shared__ int s_pos[kRopeTok];
    const int t0 = blockIdx.x * a.tok, nt = min(a.tok, a.n - t0);
    const int rot = a.plan.rotary_dim, half = rot / 2, D = a.plan.head_dim;
    const bool inter = a.plan.layout == DM_ROPE_INTERLEAVED;
    const int pu = half / VEC, units = pu + (D - rot) / VEC;
    const int total = (a.heads[0] + a.heads[1]) * units;
    bool ready = false;
    for (int base = 0; base < total; base += blockDim.x) {
        const int u = base + threadIdx.x;
        const bool live = u < total;
        int h = live ? u / units : 0;
        const int unit = u - h * units;
        const int w = h >= a.heads[0];
        if (w) h -= a.heads[0];
        const T* x = static_cast<const T*>(a.x[w]) + static_cast<int64_t>(t0) * a.x_rs[w] + h * a.x_hs[w];
        T* y = static_cast<T*>(a.y[w]) + static_cast<int64_t>(t0) * a.y_rs[w] + h * a.y_hs[w];
        const bool turn = unit < pu;
        const bool work = live && (turn || !a.inplace[w]);
        const int j0 = unit * VEC;
        const int e0 = !turn ? rot + (unit - pu) * VEC : inter ? 2 * j0 : j0, e1 = inter ? 2 * j0 + VEC : j0 + half;
        for (int tb = 0; tb < nt; tb += kRopeBatch) {
            RopeVec<T, VEC> r0[kRopeBatch], r1[kRopeBatch];
            if (work) {
#pragma unroll
                for (int i = 0; i < kRopeBatch; ++i)
                    if (tb + i < nt) {
                        r0[i].load(x + (tb + i) * a.x_rs[w] + e0);
                        if (turn) r1[i].load(x + (tb + i) * a.x_rs[w] + e1);
                    }
            }
            if (!ready) {  // every thread of the CTA passes here in its first round
                ready = true;
                for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
                    const int t = i / half, j = i - t * half;
                    const int pos = a.positions[t0 + t];
                    if (j == 0) s_pos[t] = pos;
                    const double ang = static_cast<double>(pos) * a.plan.freq[j];
                    const double red = fma(-rint(ang * 0.15915494309189535), 6.283185307179586, ang);
                    const float hi = static_cast<float>(red), lo = static_cast<float>(red - static_cast<double>(hi));
                    float s, c;
                    sincosf(hi, &s, &c);
                    cs[t][j % VEC * pu + j / VEC] =
                        make_float2((c - s * lo) * a.plan.mscale, (s + c * lo) * a.plan.mscale);
                }
                __syncthreads();
            }
            if (!work) continue;
#pragma unroll
            for (int i = 0; i < kRopeBatch; ++i) {
                const int t = tb + i;
                if (t >= nt || s_pos[t] < 0) continue;
                if (turn) {
                    float p[VEC], q[VEC];
                    r0[i].unpack(p);
                    r1[i].unpack(q);
                    if (!inter || VEC == 1) {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            const float2 f = cs[t][k * pu + unit];
                            const float v = p[k], z = q[k];
                            p[k] = v * f.x - z * f.y;
                            q[k] = z * f.x + v * f.y;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < VEC / 2; ++k) {
                            const float2 f = cs[t][k * pu + unit], g = cs[t][(VEC / 2 + k) * pu + unit];
                            float v = p[2 * k], z = p[2 * k + 1];
                            p[2 * k] = v * f.x - z * f.y;
                            p[2 * k + 1] = z * f.x + v * f.y;
                            v = q[2 * k], z = q[2 * k + 1];
                            q[2 * k] = v * g.x - z * g.y;
                            q[2 * k + 1] = z * g.x + v * g.y;
                        }
                    }
                    r0[i].pack(p);
                    r1[i].pack(q);
                    r1[i].store(y + t * a.y_rs[w] + e1);
                }
                r0[i].store(y + t * a.y_rs[w] + e0);
            }
        }
    }
}

// ---- quantising append ----------------------------------------------------------------------
// A run is the rows of one call that fall into one page.  One CTA quantises a run of one kv
// head's K or V: all its rows in registers, the largest magnitude over the CTA, then the
// codes; the page's older codes are touched only when the scale grows.  Bound by the bytes for
// prompts, read once (bf16 rows stay packed, 48 registers at D = 256 where fp32 copies took 64 and
// 20.5 us): 17.5 k tokens of 2 heads of 256 take 15.5 us, 13.2 us with the rows partly in L2, against
// 8.3 us for the bytes; the difference is the launch and one chain of slot, load, maximum, barrier, store.
// 64 single tokens take 2.3 us in a graph, that chain alone.
struct Kv8AppendArgs {
    uint8_t* pages;
    float* scales;
    const void* x[2];
    int64_t rs[2], hs[2];
    const int* slots;
    uint32_t* err;
    int n, Hkv, num_pages, window, vec;
};

constexpr int kAppendThreads = 128;

// 2^k as a float, k in [-126, 127]
DM_DEV float exp2i(int k) { return __int_as_float((k + 127) << 23); }

// smallest k in range with amax <= 448 * 2^k: 448 = 1.75 * 2^8 against amax = m 2^e, m in [1, 2)
DM_DEV int kv8_scale_exp(float amax) {
    const int b = __float_as_int(amax);
    const int k = (b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000 ? 1 : 0);
    return max(kKv8MinExp, min(kKv8MaxExp, k));
}

DM_DEV uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
DM_DEV float2 e4m3x2_to_float2(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
    return __half22float2(__half2(h));
}

// 8 consecutive elements of a row as loaded (bf16 stays packed: half the registers), and as floats
template <typename T>
struct Row8 {
    uint4 u[sizeof(T) / 2];
    DM_DEV void load(const T* p, int vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
                u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        } else {
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
            memcpy(u, e, sizeof e);
        }
    }
    DM_DEV void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
            const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 2) v[2 * j] = bf16lo(w[j]), v[2 * j + 1] = bf16hi(w[j]);
                else v[4 * i + j] = __uint_as_float(w[j]);
            }
        }
    }
};

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a) {
    constexpr int kLanes = D / 8;                   // threads of a row
    constexpr int kRows = kAppendThreads / kLanes;  // rows of a pass
    constexpr int kPasses = kKv8Page / kRows;
    __shared__ float s_max[kAppendThreads / 32];
    const int kv = blockIdx.y & 1, h = blockIdx.y >> 1, tid = threadIdx.x;
    const int row = tid / kLanes, col = (tid % kLanes) * 8;
    const T* x = static_cast<const T*>(a.x[kv]) + h * a.hs[kv] + col;
    // lane l of every warp holds slot w0 - 1 + l: the window's rows are lanes 1 .. window, the
    // lanes behind them the rest of the last run
    const int w0 = blockIdx.x * a.window, lane = tid & 31;
    const int at = w0 - 1 + lane;
    const int slot_l = at >= 0 && at < a.n ? a.slots[at] : -1;
    const int prev_l = __shfl_up_sync(0xffffffffu, slot_l, 1);
    const bool same = lane > 0 && slot_l >= 0 && prev_l >= 0 && slot_l / kKv8Page == prev_l / kKv8Page;
    const bool lead = lane > 0 && lane <= a.window && slot_l >= 0 && !same;
    const unsigned follows = __ballot_sync(0xffffffffu, same && slot_l == prev_l + 1);
    unsigned leads = __ballot_sync(0xffffffffu, lead);
    if (same && slot_l != prev_l + 1 && lane <= a.window && tid < 32) raise_error(a.err, DM_DEVERR_RANGE);
    while (leads) {
        const int l = __ffs(leads) - 1;
        leads &= leads - 1;
        const int slot = __shfl_sync(0xffffffffu, slot_l, l);
        const int page = slot / kKv8Page, off = slot % kKv8Page;
        // rows that follow slot by slot
        const unsigned rest = l < 31 ? ~(follows >> (l + 1)) : ~0u;
        const int len = __ffs(rest);
        const int t0 = w0 - 1 + l;
        if (page >= a.num_pages) {
            if (tid == 0) raise_error(a.err, DM_DEVERR_PAGE);
            continue;
        }
        Row8<T> rows[kPasses];
        float amax = 0.0f;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int r = i * kRows + row;
            if (r < len) {
                rows[i].load(x + static_cast<int64_t>(t0 + r) * a.rs[kv], a.vec);
            }
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            if (i * kRows + row < len) {
                float f[8];
                rows[i].get(f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float m = fabsf(f[e]);
                    if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
                    else odd = true;
                }
            }
        }
        if (odd) raise_error(a.err, DM_DEVERR_NONFINITE);
        amax = warp_max(amax);
        const size_t blk = (static_cast<size_t>(page) * 2 + kv) * a.Hkv + h;
        const float held = off > 0 ? a.scales[blk] : 0.0f;
        if ((tid & 31) == 0) s_max[tid >> 5] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        const int want = kv8_scale_exp(amax);
        int k = want;
        uint8_t* dst = a.pages + blk * (kKv8Page * D) + col;
        if (off > 0) {
            const int ko = max(kKv8MinExp, min(kKv8MaxExp, ((__float_as_int(held) >> 23) & 0xff) - 127));
            k = max(want, ko);
            if (k > ko) {
                const float ratio = k - ko > 126 ? 0.0f : exp2i(ko - k);
                for (int r = row; r < off; r += kRows) {
                    uint2* p = reinterpret_cast<uint2*>(dst + r * D);
                    uint2 c = *p;
                    uint32_t* cw = &c.x;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 f = e4m3x2_to_float2(cw[j]), g = e4m3x2_to_float2(cw[j] >> 16);
                        cw[j] = e4m3x4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
                    }
                    *p = c;
                }
            }
        }
        const float inv = exp2i(-k);
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int r = i * kRows + row;
            if (r < len) {
                float f[8];
                rows[i].get(f);
                *reinterpret_cast<uint2*>(dst + (off + r) * D) =
                    make_uint2(e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                               e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
            }
        }
        if (tid == 0) a.scales[blk] = exp2i(k);
        __syncthreads();
    }
}

template <typename T>
static cudaError_t launch_append(const Kv8AppendArgs& a, int D, cudaStream_t s) {
    const dim3 grid((a.n + a.window - 1) / a.window, 2 * a.Hkv);
    if (D == 64) kv8_append_kernel<T, 64><<<grid, kAppendThreads, 0, s>>>(a);
    else if (D == 128) kv8_append_kernel<T, 128><<<grid, kAppendThreads, 0, s>>>(a);
    else kv8_append_kernel<T, 256><<<grid, kAppendThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace dm

using namespace dm;

extern "C" int32_t dm_kv8_status(uint32_t* err_dev, void* stream, char* eb, uint64_t es) {
    const char* st = "kv8_status";
    if (eb && es > 0) eb[0] = '\0';
    Kv8Device g;
    if (!err_dev) {
        int dev = -1;
        if (cudaGetDevice(&dev) == cudaSuccess) err_dev = kv8_error_word(nullptr, dev);
        if (!err_dev) return kv8_err(eb, es, DM_ERR_CUDA, "CUDA_ERROR", st, "no device");
    }
    if (int rc = g.enter(err_dev, st, eb, es)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(s, &cap);
    if (e != cudaSuccess || cap != cudaStreamCaptureStatusNone)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "the stream is being captured");
    uint32_t w = 0;
    e = cudaMemcpyAsync(&w, err_dev, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && w) e = cudaMemsetAsync(err_dev, 0, 4, s);
    if (e != cudaSuccess) return kv8_err(eb, es, DM_ERR_CUDA, "CUDA_ERROR", st, "%s", cudaGetErrorString(e));
    if (w & DM_DEVERR_TIMEOUT)
        return kv8_err(eb, es, DM_ERR_TIMEOUT, "DEVICE_TIMEOUT", st, "a bounded device wait ran out (word 0x%x)", w);
    if (w & DM_DEVERR_CAPACITY)
        return kv8_err(eb, es, DM_ERR_CAPACITY, "CAPACITY_ERROR", st,
                       "pages, table width or token buffers do not suffice (word 0x%x)", w);
    if (w & (DM_DEVERR_PAGE | DM_DEVERR_RANGE))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st,
                       "a page id, slot, length or row range out of contract (word 0x%x)", w);
    if (w) return kv8_err(eb, es, DM_ERR_NONFINITE, "NONFINITE_ERROR", st, "non-finite values (word 0x%x)", w);
    return DM_OK;
}

extern "C" int32_t dm_kv8_plan(int32_t n, const int32_t* ctx_lens, const int32_t* new_lens, int32_t* block_table,
                               int32_t table_width, int32_t* free_pages, int32_t free_capacity,
                               const int32_t* free_state, int32_t* free_state_out, int32_t* seq_lens, int32_t* cu_new,
                               int32_t max_tokens, int32_t* slots, int32_t* positions, int32_t* requests,
                               uint32_t* err_dev, void* stream, char* eb, uint64_t es) {
    const char* st = "kv8_plan";
    if (eb && es > 0) eb[0] = '\0';
    if (!ctx_lens || !new_lens || !block_table || !free_pages || !free_state || !free_state_out || !seq_lens ||
        !cu_new || !slots || !positions || !requests)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    if (n < 1 || n > DM_KV8_MAX_REQUESTS || table_width < 1 ||
        static_cast<int64_t>(n) * table_width > (1 << 27) || free_capacity < 1 || free_capacity >= (1 << 27) ||
        max_tokens < 1 || max_tokens > (1 << 30))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st,
                       "need 1 <= n <= %d, 1 <= table_width, n * table_width <= 2^27, 1 <= free_capacity < 2^27, "
                       "1 <= max_tokens <= 2^30 (n=%d, width=%d, capacity=%d, max_tokens=%d)",
                       DM_KV8_MAX_REQUESTS, n, table_width, free_capacity, max_tokens);
    Kv8Device g;
    if (int rc = g.enter(ctx_lens, st, eb, es)) return rc;
    Kv8PlanArgs a{};
    a.ctx = ctx_lens;
    a.add = new_lens;
    a.table = block_table;
    a.free_pages = free_pages;
    a.state = free_state;
    a.state_out = free_state_out;
    a.seq_lens = seq_lens;
    a.cu_new = cu_new;
    a.slots = slots;
    a.positions = positions;
    a.requests = requests;
    a.err = kv8_error_word(err_dev, g.dev);
    a.n = n;
    a.width = table_width;
    a.cap = free_capacity;
    a.max_tokens = max_tokens;
    a.in_place = seq_lens == ctx_lens || free_state_out == free_state;
    const int work = max_tokens > n ? max_tokens : n;
    const int block = work <= 256 ? 256 : 1024;
    // CTAs by the entries to write: the tokens', and the pages that requests may give back
    int grid = ((max_tokens > 4 * n ? max_tokens : 4 * n) + 1023) / 1024;
    if (grid > g.num_sms) grid = g.num_sms;
    // lengths in place, the count not: no word of free_state_out is known to be zero, so one CTA
    if (seq_lens == ctx_lens && free_state_out != free_state) grid = 1;
    const size_t smem = 3 * static_cast<size_t>(n + 1) * sizeof(unsigned);
    cudaError_t e = cudaSuccess;
    if (smem > 40 * 1024) {
        // once per device and for the largest plan: the limit is the function's, calls on other threads share it
        static std::atomic<bool> ready[64];
        if (g.dev >= 64 || !ready[g.dev].load(std::memory_order_relaxed)) {
            e = cudaFuncSetAttribute(kv8_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     3 * (DM_KV8_MAX_REQUESTS + 1) * static_cast<int>(sizeof(unsigned)));
            if (e == cudaSuccess && g.dev < 64) ready[g.dev].store(true, std::memory_order_relaxed);
        }
    }
    if (e == cudaSuccess) {
        kv8_plan_kernel<<<grid, block, smem, static_cast<cudaStream_t>(stream)>>>(a);
        e = cudaGetLastError();
    }
    return launch_status(e, st, eb, es);
}

extern "C" int32_t dm_rope_plan_init(const dm_rope_params* p, dm_rope_plan* plan, char* eb, uint64_t es) {
    const char* st = "rope_plan";
    if (eb && es > 0) eb[0] = '\0';
    if (!p || !plan) return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    const int r = p->rotary_dim, D = p->head_dim;
    if (D < 16 || D > 256 || D % 8 != 0 || r < 16 || r > D || r % 16 != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", st,
                       "need head_dim a multiple of 8 up to 256 and rotary_dim a multiple of 16 up to it (%d, %d)", D,
                       r);
    if ((p->layout != DM_ROPE_HALF && p->layout != DM_ROPE_INTERLEAVED) || p->scaling < DM_ROPE_NONE ||
        p->scaling > DM_ROPE_YARN)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", st, "unknown layout or scaling");
    if (!(p->theta > 1.0) || !std::isfinite(p->theta))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", st, "need a finite theta > 1");
    if (p->scaling != DM_ROPE_NONE && (!(p->factor >= 1.0) || !std::isfinite(p->factor)))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", st, "need a finite factor >= 1");
    if (p->scaling == DM_ROPE_YARN && (!(p->original_context > 0.0) || !std::isfinite(p->original_context) ||
                                       !(p->beta_slow > 0.0) || !(p->beta_fast > p->beta_slow) ||
                                       !std::isfinite(p->beta_fast) || !std::isfinite(p->attention_factor)))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", st,
                       "need original_context > 0 and beta_fast > beta_slow > 0");
    *plan = dm_rope_plan{};
    plan->head_dim = D;
    plan->rotary_dim = r;
    plan->layout = p->layout;
    plan->mscale = 1.0f;
    double lo = 0.0, hi = 0.0;
    if (p->scaling == DM_ROPE_YARN) {
        const double two_pi = 6.283185307179586, den = 2.0 * std::log(p->theta);
        lo = std::fmax(std::floor(r * std::log(p->original_context / (p->beta_fast * two_pi)) / den), 0.0);
        hi = std::fmin(std::ceil(r * std::log(p->original_context / (p->beta_slow * two_pi)) / den), r - 1.0);
        plan->mscale = static_cast<float>(p->attention_factor > 0.0 ? p->attention_factor
                                                                    : 0.1 * std::log(p->factor) + 1.0);
    }
    for (int i = 0; i < r / 2; ++i) {
        const double f = std::pow(p->theta, -2.0 * i / r);
        double g = 0.0;
        if (p->scaling == DM_ROPE_LINEAR) g = 1.0;
        if (p->scaling == DM_ROPE_YARN) g = std::fmin(std::fmax((i - lo) / std::fmax(hi - lo, 0.001), 0.0), 1.0);
        plan->freq[i] = g == 0.0 ? f : f * (1.0 - g) + f / p->factor * g;
    }
    return DM_OK;
}

extern "C" int32_t dm_rope(const dm_rope_plan* plan, int32_t dtype, int32_t n, const int32_t* positions, const void* q,
                           int64_t q_rs, int64_t q_hs, void* qo, int64_t qo_rs, int64_t qo_hs, int32_t Hq,
                           const void* k, int64_t k_rs, int64_t k_hs, void* ko, int64_t ko_rs, int64_t ko_hs,
                           int32_t Hk, void* stream, char* eb, uint64_t es) {
    const char* st = "rope";
    if (eb && es > 0) eb[0] = '\0';
    if (!plan || plan->head_dim < 16 || plan->head_dim > 256 || plan->head_dim % 8 != 0 || plan->rotary_dim < 16 ||
        plan->rotary_dim > plan->head_dim || plan->rotary_dim % 16 != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "no plan of dm_rope_plan_init");
    if (dtype != DM_DTYPE_BF16 && dtype != DM_DTYPE_F32)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "dtype is bf16 or fp32");
    if (n < 0 || n > (1 << 30) || Hq < 0 || Hk < 0 || Hq > 65536 || Hk > 65536)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "n: 0 to 2^30, head counts: 0 to 65536");
    if (n == 0 || Hq + Hk == 0) return DM_OK;
    if (!positions || (Hq && (!q || !qo)) || (Hk && (!k || !ko)))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    Kv8Device g;
    if (int rc = g.enter(positions, st, eb, es)) return rc;
    const int elem = dtype == DM_DTYPE_F32 ? 4 : 2;
    RopeArgs a{};
    a.plan = *plan;
    a.x[0] = q, a.x_rs[0] = q_rs, a.x_hs[0] = q_hs, a.y[0] = qo, a.y_rs[0] = qo_rs, a.y_hs[0] = qo_hs;
    a.x[1] = k, a.x_rs[1] = k_rs, a.x_hs[1] = k_hs, a.y[1] = ko, a.y_rs[1] = ko_rs, a.y_hs[1] = ko_hs;
    a.heads[0] = Hq, a.heads[1] = Hk;
    a.positions = positions;
    a.n = n;
    bool vec = true;
    for (int i = 0; i < 2; ++i) {
        if (!a.heads[i]) continue;
        if (a.x[i] == a.y[i]) {
            if (a.x_rs[i] != a.y_rs[i] || a.x_hs[i] != a.y_hs[i])
                return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "in place needs the same strides");
            a.inplace[i] = 1;
        }
        vec = vec && kv8_aligned(a.x[i], a.x_rs[i], a.x_hs[i], elem, 16) &&
              kv8_aligned(a.y[i], a.y_rs[i], a.y_hs[i], elem, 16);
    }
    // few tokens: a CTA each, for the shortest wait; many: 8, whose angles are then computed by
    // the CTA's threads in one round
    a.tok = n <= 8 * g.num_sms ? 1 : kRopeTok;
    const int grid = (n + a.tok - 1) / a.tok;
    // threads: the units of a token in equal rounds
    const int v = vec ? 16 / elem : 1;
    const int total = (Hq + Hk) * ((plan->head_dim - plan->rotary_dim / 2) / v);
    const int rounds = (total + 383) / 384;
    const int block = ((total + rounds - 1) / rounds + 31) / 32 * 32;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == DM_DTYPE_F32) {
        if (vec) rope_kernel<float, 4><<<grid, block, 0, s>>>(a);
        else rope_kernel<float, 1><<<grid, block, 0, s>>>(a);
    } else {
        if (vec) rope_kernel<__nv_bfloat16, 8><<<grid, block, 0, s>>>(a);
        else rope_kernel<__nv_bfloat16, 1><<<grid, block, 0, s>>>(a);
    }
    return launch_status(cudaGetLastError(), st, eb, es);
}

extern "C" int32_t dm_kv8_append(const dm_kv8_cache* c, int32_t dtype, int32_t n, const void* k, int64_t k_rs,
                                 int64_t k_hs, const void* v, int64_t v_rs, int64_t v_hs, const int32_t* slots,
                                 uint32_t* err_dev, void* stream, char* eb, uint64_t es) {
    const char* st = "kv8_append";
    if (eb && es > 0) eb[0] = '\0';
    if (int rc = kv8_check_cache(c, st, eb, es)) return rc;
    if (dtype != DM_DTYPE_BF16 && dtype != DM_DTYPE_F32)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "dtype is bf16 or fp32");
    if (n < 0 || n > (1 << 30)) return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "n = %d", n);
    if (n == 0) return DM_OK;
    if (!k || !v || !slots) return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    Kv8Device g;
    if (int rc = g.enter(c->pages, st, eb, es)) return rc;
    const int elem = dtype == DM_DTYPE_F32 ? 4 : 2;
    Kv8AppendArgs a{};
    a.pages = c->pages;
    a.scales = c->scales;
    a.x[0] = k, a.rs[0] = k_rs, a.hs[0] = k_hs;
    a.x[1] = v, a.rs[1] = v_rs, a.hs[1] = v_hs;
    a.slots = slots;
    a.err = kv8_error_word(err_dev, g.dev);
    a.n = n;
    a.Hkv = c->num_kv_heads;
    a.num_pages = c->num_pages;
    // rows of a CTA: one when the rows may all be in pages of their own (a decode step), more
    // for prompts, where a CTA per row would mostly find that an earlier one has its page.  us with 1 /
    // 4 / 16 rows, cold, 2 heads of 256 in bf16: 500 single tokens 8 / 10 / 23, 2000 16 / 16 / 24, 2000 of
    // prompts 10 / 8 / 10; 3000 single 21 / 21 / 25, 8000 45 / 39 / 43, 7000 of prompts 23 / 12 / 14;
    // 9000 27 / 14 / 14, 17000 42 / 23 / 18
    a.window = n <= 2048 ? 1 : n <= 8192 ? 4 : 16;
    a.vec = kv8_aligned(k, k_rs, k_hs, elem, 16) && kv8_aligned(v, v_rs, v_hs, elem, 16);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == DM_DTYPE_F32 ? launch_append<float>(a, c->head_dim, s)
                                                : launch_append<__nv_bfloat16>(a, c->head_dim, s);
    return launch_status(e, st, eb, es);
}
