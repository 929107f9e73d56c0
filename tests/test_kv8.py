"""The 8-bit paged KV cache operators (slot planning, rotary positions, quantised append,
attention over the cache) against plain implementations in 64 bits."""
import ctypes as C
import json
import math

import numpy as np
import pytest
import torch

from disk_streaming_moe_engine_b200 import DmError, _lib, kv8

PAGE = 16
F32_STEP, BF16_STEP = 2.0 ** -24, 2.0 ** -8  # largest relative rounding (half a step)
DEV = "cuda"


# ---- plain forms ------------------------------------------------------------------------------

def plain_plan(free, count, table, ctx, new, max_tokens):
    """Lists and loops: (refused, seq_lens, cu_new, slots, positions, requests, table, free, count)."""
    n, width = table.shape
    table, free = table.copy(), free.copy()
    have = [-(-c // PAGE) for c in ctx]
    need = [0 if w < 0 else -(-(c + w) // PAGE) for c, w in zip(ctx, new)]
    stack = list(free[:count]) + [table[i, p] for i in range(n) if new[i] < 0 for p in range(have[i])]
    grow = sum(need[i] - have[i] for i in range(n) if new[i] >= 0)
    total = sum(max(w, 0) for w in new)
    none = np.full(max_tokens, -1, np.int32)
    if (any(max(a, b) > width for a, b in zip(need, have)) or grow > len(stack) or len(stack) > len(free)
            or total > max_tokens or any(c < 0 for c in ctx) or any(w < -1 for w in new)):
        return True, list(ctx), [0] * (n + 1), none, none.copy(), none.copy(), table, free, count
    slots, pos, req = none, none.copy(), none.copy()
    t, cu = 0, [0]
    for i in range(n):
        if new[i] >= 0:
            for p in range(have[i], need[i]):
                table[i, p] = stack.pop()
            for x in range(ctx[i], ctx[i] + new[i]):
                slots[t], pos[t], req[t] = table[i, x // PAGE] * PAGE + x % PAGE, x, i
                t += 1
        cu.append(t)
    if len(stack) > count:
        free[count:len(stack)] = stack[count:]
    return False, [0 if w < 0 else c + w for c, w in zip(ctx, new)], cu, slots, pos, req, table, free, len(stack)


def e4m3_values():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b & 128, -v, v)


E4M3 = e4m3_values()


def to_e4m3(x):
    """Codes of the nearest values, ties to the even code, beyond 448 the largest; NaN 0x7f."""
    pos = E4M3[:127]
    a = np.minimum(np.abs(x), 448.0)
    hi = np.clip(np.searchsorted(pos, np.nan_to_num(a)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = pos[hi] - a, a - pos[lo]
    c = np.where((up < down) | ((up == down) & (hi % 2 == 0)) | (a >= pos[hi]), hi, lo)
    c = np.where(np.isnan(x), 127, c)
    return (c | np.where(np.signbit(x) & ~np.isnan(x), 128, 0)).astype(np.uint8)


def plain_append(pages, scales, k, v, slots):
    pages, scales = pages.copy(), scales.astype(np.float64)
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        page, off = divmod(int(slots[t]), PAGE)
        e = t
        while e < len(slots) and slots[e] // PAGE == page and slots[e] >= 0:
            e += 1
        for c, x in enumerate((k, v)):
            for h in range(x.shape[1]):
                new = x[t:e, h].astype(np.float64)
                fin = np.abs(new[np.isfinite(new)])
                top = fin.max() if fin.size else 0.0
                want = 2.0 ** -100 if top <= 448 * 2.0 ** -100 else 2.0 ** min(100, math.ceil(round(math.log2(top / 448), 13)))
                assert top <= 448 * want or want == 2.0 ** 100
                s = want
                if off:
                    s = max(want, scales[page, c, h])
                    pages[page, c, h, :off] = np.where(
                        s > scales[page, c, h], to_e4m3(E4M3[pages[page, c, h, :off]] * (scales[page, c, h] / s)),
                        pages[page, c, h, :off])
                scales[page, c, h] = s
                pages[page, c, h, off:off + e - t] = to_e4m3(new / s)
        t = e
    return pages, scales


def plain_attention(cache, q, table, lens, cu, scale):
    """64-bit results, their magnitudes (sum p |v|, and the row's largest p sV times the sum of
    |codes|), the largest sum |q k| of every row, lse: elementary operations, one request at a
    time."""
    dev, f64 = cache.device, torch.float64
    q = q.double()
    grp = q.shape[1] // cache.num_kv_heads
    value = torch.from_numpy(E4M3).to(dev)
    out, mag, small = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    sat = torch.zeros(q.shape[:2], dtype=f64, device=dev)
    lse = torch.full(q.shape[:2], -math.inf, dtype=f64, device=dev)
    for i, n in enumerate(lens):
        m = int(cu[i + 1] - cu[i])
        if not m or not n:
            continue
        pos = torch.arange(n, device=dev)
        ids = torch.from_numpy(np.asarray(table[i], np.int64)).to(dev)[pos // PAGE]
        codes = value[cache.pages[ids, :, :, pos % PAGE].long()]  # [n][2][hk][d]
        sc = cache.scales[ids].double()
        see = pos[None, :] < (n - m + torch.arange(m, device=dev) + 1)[:, None]  # [m][n]
        some = see.any(1)
        rows = slice(int(cu[i]), int(cu[i + 1]))
        for h in range(cache.num_kv_heads):
            hs = slice(h * grp, (h + 1) * grp)
            k, cv, sv = codes[:, 0, h] * sc[:, 0, h, None], codes[:, 1, h], sc[:, 1, h]
            v = torch.where(see.any(0)[:, None], cv * sv[:, None], 0.0)
            x = q[rows, hs]
            s = torch.where(see[:, None], x @ k.T * scale, -math.inf)  # [m][grp][n]
            top = s.amax(-1, keepdim=True).clamp(min=-1e300)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            p = p / total.clamp(min=1e-300)
            lse[rows, hs] = torch.where(some[:, None], (top + torch.log(total))[..., 0], -math.inf)
            out[rows, hs], mag[rows, hs] = p @ v, p @ v.abs()
            small[rows, hs] = (p * sv).amax(-1, keepdim=True) * (see.double() @ cv.abs().nan_to_num())[:, None]
            sat[rows, hs] = torch.where(see[:, None], x.abs() @ k.abs().T, 0.0).amax(-1) * abs(scale)
    return out.cpu().numpy(), (mag.cpu().numpy(), small.cpu().numpy()), sat.cpu().numpy(), lse.cpu().numpy()


def attention_tolerance(out, mag, sat, d, keys, dtype, rows=1):
    """A score is a sum over D / 16 chained products of 16 terms, each at most 2^-22 of the sum
    of magnitudes off, of q split to 22 bits (fp32) or, in the tile kernel, to 2^-17 of the
    row's largest element; an error e of every score changes an output by at most
    2 e sum p |v|.  Weights: 2^-20 (two fp16 terms, or fp32) per key page of the running sum;
    bf16 outputs carry weights of at least 8 bits and their own rounding.  The 8 bits are two
    e4m3 terms, the second scaled by 2^4, of 64 times the weight (relative to the row's
    largest, at least 2^-2 of it): its smallest step is 2^-9 / 2^4 / 2^6, so a weight is off by
    2^-20 of the largest one's p sV at least, on a code of V.  From 40 query rows per request and
    kv head on, the second term may have the scale of the first: 2^-16."""
    mag, small = mag
    ds = sat[..., None] * (d / 16 + 1) * 2.0 ** -22
    tol = (2 * ds + (keys / PAGE + 4) * 2.0 ** -22 + 2.0 ** -20) * mag
    if dtype == torch.bfloat16:
        tol = tol + BF16_STEP * np.abs(out) + (BF16_STEP + 2 * sat[..., None] * 2.0 ** -13) * mag + (2.0 ** -16 if rows >= 40 else 2.0 ** -18) * small
    return tol + 1e-30


# ---- inputs -----------------------------------------------------------------------------------

def make_cache(n_pages, hk, d, seed, lo=-9, hi=-5):
    g = np.random.default_rng(seed)
    x = torch.randn((n_pages, 2, hk, PAGE, d), generator=torch.Generator(DEV).manual_seed(seed), device=DEV)
    codes = x.mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = np.exp2(g.integers(lo, hi + 1, (n_pages, 2, hk)).astype(np.float64)).astype(np.float32)
    return kv8.Kv8Cache(codes, torch.from_numpy(scales).to(DEV))


def make_table(lens, n_pages, seed, extra=0, width=None):
    g = np.random.default_rng(seed + 1)
    need = [-(-n // PAGE) for n in lens]
    perm = g.permutation(n_pages)
    table = np.full((len(lens), width or max(max(need) + extra, 1)), -7, np.int32)  # unused entries are garbage
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        at += k
    return table


def dev32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def check_attention(lens, rows, hk, grp, d, dtype, seed=0, scale=None, cu_none=False, mutate=None, extra=0):
    n_pages = sum(-(-n // PAGE) for n in lens) + 3
    cache = make_cache(n_pages, hk, d, seed)
    table = make_table(lens, n_pages, seed, extra)
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = torch.randn(int(cu[-1]), hk * grp, d, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)
    if mutate:
        mutate(cache, table, q)
    scale = d ** -0.5 if scale is None else scale
    err = kv8.error_word()
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = kv8.attention(cache, q, dev32(table), dev32(lens), None if cu_none else dev32(cu), max(max(rows), 1),
                        sm_scale=scale, lse=lse, workspace=kv8.attention_workspace(cache), err=err)
    kv8.check(err)
    out, mag, sat, want_lse = plain_attention(cache, q, table, lens, cu, scale)
    tol = attention_tolerance(out, mag, sat, d, max(lens), dtype, max(rows) * grp)
    diff = np.abs(got.double().cpu().numpy() - out)
    assert (diff <= tol).all(), (diff / tol).max()
    finite = np.isfinite(want_lse)
    got_lse = lse.double().cpu().numpy()
    assert (np.isneginf(got_lse) == ~finite).all()
    soft = 2.0 ** -12 if dtype == torch.bfloat16 else (d / 16 + 1) * 2.0 ** -22
    off = np.abs(got_lse[finite] - want_lse[finite])
    assert (off <= (sat * soft + np.abs(want_lse) * 2.0 ** -22 + 2.0 ** -18)[finite]).all()
    return cache, table, cu, q, got


# ---- CPU: refusals and host-side plans ----------------------------------------------------------

def _call(lib, name, *args):
    buf = C.create_string_buffer(512)
    rc = getattr(lib, name)(*args, buf, 512)
    return rc, json.loads(buf.value.decode()) if buf.value else None


def _fake_cache(**kw):
    f = dict(pages=1 << 20, scales=1 << 21, num_pages=4, num_kv_heads=2, head_dim=128, reserved=0)
    f.update(kw)
    return _lib.DmKv8Cache(*f.values())


@pytest.mark.parametrize("kw", [dict(pages=None), dict(scales=None), dict(head_dim=96), dict(num_pages=0),
                                dict(num_kv_heads=0), dict(pages=(1 << 20) + 8), dict(reserved=1),
                                dict(num_pages=1 << 26, num_kv_heads=8)])
def test_cache_refusals(lib, kw):
    c = _fake_cache(**kw)
    one = 1 << 22  # never dereferenced: the checks come first
    rc, err = _call(lib, "dm_kv8_append", C.addressof(c), 0, 1, one, 0, 0, one, 0, 0, one, None, None)
    assert rc == _lib.DM_ERR_INVALID_ARG and set(err) == {"error_type", "detail", "stage", "layer"}
    a = _lib.DmKv8AttnArgs()
    rc, err = _call(lib, "dm_kv8_attention", C.addressof(c), C.addressof(a), None)
    assert rc == _lib.DM_ERR_INVALID_ARG and err["stage"] == "kv8_attention"


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(n=-1), dict(rows=-1), dict(num_q_heads=3), dict(num_q_heads=0),
                                dict(sm_scale=float("nan")), dict(table_width=0), dict(table_width=(1 << 26) + 1), dict(max_q_len=0),
                                dict(max_q_len=2), dict(rows=3), dict(reserved=1), dict(q=None), dict(out=None),
                                dict(block_table=None), dict(seq_lens=None), dict(workspace=None),
                                dict(workspace=(1 << 22) + 16)])
def test_attention_refusals(lib, kw):
    c, one = _fake_cache(), 1 << 22
    f = dict(dtype=0, n=4, num_q_heads=8, max_q_len=1, rows=4, table_width=9, sm_scale=0.1, reserved=0, q=one,
             q_row_stride=1024, q_head_stride=128, out=one, out_row_stride=1024, out_head_stride=128, lse=None,
             block_table=one, seq_lens=one, cu_q=None, workspace=one, workspace_bytes=1 << 40, err_dev=None)
    f.update(kw)
    a = _lib.DmKv8AttnArgs(*f.values())
    rc, _ = _call(lib, "dm_kv8_attention", C.addressof(c), C.addressof(a), None)
    assert rc == _lib.DM_ERR_INVALID_ARG


def test_size_refusals(lib):
    """Counts whose products would pass 32 bits in the kernels."""
    c, one = _fake_cache(), 1 << 22
    a = _lib.DmKv8AttnArgs(dtype=0, n=1, num_q_heads=1 << 11, max_q_len=1, rows=1 << 20, table_width=1, sm_scale=0.1,
                           q=one, out=one, block_table=one, seq_lens=one, workspace=one, workspace_bytes=1 << 40)
    rc, err = _call(lib, "dm_kv8_attention", C.addressof(c), C.addressof(a), None)
    assert rc == _lib.DM_ERR_INVALID_ARG and "2^31" in err["detail"]
    plan = kv8.RopePlan(64)
    for n, hq in (((1 << 30) + 1, 1), (1, 65537), (-1, 1)):
        rc, err = _call(lib, "dm_rope", plan._ref, 0, n, one, one, 64, 64, one, 64, 64, hq, None, 0, 0, None, 0, 0, 0,
                        None)
        assert rc == _lib.DM_ERR_INVALID_ARG and "2^30" in err["detail"]


def test_empty_calls_need_no_device(lib):
    c, one = _fake_cache(), 1 << 22
    assert _call(lib, "dm_kv8_append", C.addressof(c), 0, 0, one, 0, 0, one, 0, 0, one, None, None)[0] == 0
    a = _lib.DmKv8AttnArgs(dtype=0, n=0, num_q_heads=8, max_q_len=1, rows=0, table_width=1, sm_scale=1.0)
    assert _call(lib, "dm_kv8_attention", C.addressof(c), C.addressof(a), None)[0] == 0


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=8193), dict(width=0), dict(cap=0), dict(tokens=0),
                                 dict(n=8192, width=1 << 15), dict(null=True)])
def test_plan_refusals(lib, bad):
    one = 1 << 22
    p = None if bad.get("null") else one
    rc, err = _call(lib, "dm_kv8_plan", bad.get("n", 4), p, one, one, bad.get("width", 8), one, bad.get("cap", 64), one,
                    one, one, one, bad.get("tokens", 4), one, one, one, None, None)
    assert rc == _lib.DM_ERR_INVALID_ARG and err["stage"] == "kv8_plan"


@pytest.mark.parametrize("kw", [dict(head_dim=260), dict(head_dim=12), dict(rotary_dim=8), dict(rotary_dim=24),
                                dict(rotary_dim=144), dict(theta=1.0), dict(theta=float("inf")),
                                dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=4.0, beta_fast=1.0),
                                dict(scaling="yarn", original_context=0.0), dict(layout="spiral"),
                                dict(scaling="cubic")])
def test_rope_plan_refusals(lib, kw):
    f = dict(head_dim=128, rotary_dim=64)
    f.update(kw)
    with pytest.raises(DmError):
        kv8.RopePlan(**f)


def plain_freq(rot, theta, scaling, factor, orig=32768):
    i = np.arange(rot // 2)
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        at = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
        g = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f * (1 - g) + f / factor * g, 0.1 * math.log(factor) + 1
    return f, 1.0


@pytest.mark.parametrize("scaling", ["none", "linear", "yarn"])
@pytest.mark.parametrize("rot,theta", [(16, 1e4), (64, 1e7), (128, 5e5), (256, 1e6)])
def test_rope_plan_frequencies(lib, scaling, rot, theta):
    p = kv8.RopePlan(256, rot, theta=theta, scaling=scaling, factor=8.0)
    f, m = plain_freq(rot, theta, scaling, 8.0)
    np.testing.assert_allclose(p.freq, f, rtol=1e-13)
    assert p.mscale == np.float32(m)


def test_rope_plan_attention_factor(lib):
    assert kv8.RopePlan(64, scaling="yarn", factor=4.0, attention_factor=1.5).mscale == 1.5


def test_cache_wrapper_refusals():
    with pytest.raises(DmError):  # not on the GPU
        kv8.Kv8Cache(torch.zeros(2, 2, 1, 16, 64, dtype=torch.uint8), torch.ones(2, 2, 1))


def test_plain_e4m3_matches_torch():
    """The test's own rounding against torch's conversion, values, halves and neighbours."""
    v = E4M3[:127]
    x = np.concatenate([v, (v[1:] + v[:-1]) / 2, v * (1 + 2.0 ** -20), v * (1 - 2.0 ** -20)])
    x = np.concatenate([x, -x]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(to_e4m3(x.astype(np.float64)), want)


# ---- GPU: plan ----------------------------------------------------------------------------------

def run_plan(ctx, new, width, cap, used_pages, max_tokens, seed=0, in_place=False):
    """Runs the operator and the plain form on the same state."""
    n = len(ctx)
    perm = np.random.default_rng(seed).permutation(cap).astype(np.int32)
    table = np.full((n, width), -3, np.int32)
    at = 0
    for i, c in enumerate(ctx):
        k = min(-(-max(c, 0) // PAGE), width)
        table[i, :k] = perm[at:at + k]
        at += k
    at = max(at, used_pages)
    count = cap - at
    free = np.full(cap, -5, np.int32)
    free[:count] = perm[at:]
    want = plain_plan(free, count, table, list(ctx), list(new), max_tokens)
    d_free, d_state, d_table, d_ctx = dev32(free), dev32([count, 0]), dev32(table), dev32(ctx)
    err = kv8.error_word()
    state_out = None if in_place else dev32([-1, 0])
    out = None
    if in_place:
        tok = torch.zeros((3, max_tokens), dtype=torch.int32, device=DEV)
        out = kv8.SlotPlan(d_ctx, torch.zeros(n + 1, dtype=torch.int32, device=DEV), tok[0], tok[1], tok[2])
    p = kv8.plan_slots(d_free, d_state, d_table, d_ctx, dev32(new), max_tokens, state_out=state_out, out=out, err=err)
    refused, lens, cu, slots, pos, req, table, free, left = want
    for got, ref in zip(p, (lens, cu, slots, pos, req)):
        np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(ref, np.int32))
    np.testing.assert_array_equal(d_table.cpu().numpy(), table)
    np.testing.assert_array_equal(d_free.cpu().numpy(), free)
    np.testing.assert_array_equal((d_state if in_place else state_out).cpu().numpy(), [left, 0])
    if refused:
        with pytest.raises(DmError):
            kv8.check(err)
    kv8.check(err)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,ctx_hi,new_hi,release,pad,seed", [
    (1, 0, 1, 0.0, 0, 0), (1, 40, 1, 0.0, 0, 1), (3, 33, 0, 0.0, 5, 2), (64, 500, 1, 0.0, 0, 3),
    (65, 100, 40, 0.3, 7, 4), (257, 20, 3, 0.5, 1, 5), (1000, 60, 30, 0.1, 100, 6), (1025, 17, 2, 0.2, 0, 7),
    (8192, 40, 9, 0.2, 3, 8), (40, 3000, 2500, 0.2, 0, 9), (5, 100, 0, 1.0, 4, 10)])
def test_plan(lib, n, ctx_hi, new_hi, release, pad, seed, in_place):
    g = np.random.default_rng(seed)
    ctx, new = g.integers(0, ctx_hi + 1, n), g.integers(0, new_hi + 1, n)
    new[g.random(n) < release] = -1
    width = int((ctx + np.maximum(new, 0) + 15).max() // PAGE) + 1
    used = int(sum(-(-c // PAGE) for c in ctx))
    grow = int(sum(-(-(c + w) // PAGE) - -(-c // PAGE) for c, w in zip(ctx, new) if w >= 0))
    back = int(sum(-(-c // PAGE) for c, w in zip(ctx, new) if w < 0))
    cap = used + max(grow - back, 0) + (seed % 2) * 5  # without spare pages half of the time
    total = max(1, int(np.maximum(new, 0).sum()) + pad)
    assert not run_plan(ctx, new, width, max(cap, 1), used, total, seed, in_place)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new,width,cap,used,tokens", [
    ([16, 5], [1, 1], 4, 2, 2, 8),        # no page left
    ([16, 5], [40, 1], 3, 64, 2, 64),     # table too narrow
    ([16, 5], [20, 9], 4, 64, 2, 28),     # one token more than the buffers hold
    ([-1, 5], [1, 1], 4, 64, 1, 8),       # negative length
    ([16, 5], [-2, 1], 4, 64, 2, 8),      # unknown request kind
    ([2 ** 31 - 5, 5], [9, 1], 4, 64, 1, 16),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_all_or_nothing(lib, ctx, new, width, cap, used, tokens, in_place):
    assert run_plan(ctx, new, width, cap, used, tokens, 1, in_place)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("own_lens,own_state", [(True, False), (False, True), (False, False)])
def test_plan_partly_in_place(lib, own_lens, own_state):
    """Only the lengths, or only the state, in place, over many CTAs; a separate state's memory
    holds anything before the call."""
    n, new = 40, 700
    cap = n * 47
    free, state = kv8.free_list(cap)
    table = torch.zeros((n, 48), dtype=torch.int32, device=DEV)
    lens = dev32([30] * n)
    tok = torch.zeros((3, n * new), dtype=torch.int32, device=DEV)
    held = kv8.plan_slots(free, state, table, dev32([0] * n), lens, 30 * n)  # pages of the old tokens
    count = int(state[0])
    pages, old = free.cpu().numpy().copy(), table.cpu().numpy().copy()
    out = kv8.SlotPlan(lens if own_lens else torch.zeros_like(lens), torch.zeros(n + 1, dtype=torch.int32, device=DEV),
                       tok[0], tok[1], tok[2])
    state_out = None if own_state else dev32([-7, 1234567])
    err = kv8.error_word()
    p = kv8.plan_slots(free, state, table, lens, dev32([new] * n), n * new, state_out=state_out, out=out, err=err)
    kv8.check(err)
    refused, want_lens, cu, slots, pos, req, want_table, _, left = plain_plan(pages, count, old, [30] * n, [new] * n,
                                                                              n * new)
    assert not refused and held.seq_lens.tolist() == [30] * n
    for got, ref in zip(p, (want_lens, cu, slots, pos, req)):
        np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(ref, np.int32))
    np.testing.assert_array_equal(table.cpu().numpy(), want_table)
    assert (state if own_state else state_out).tolist() == [left, 0]


# ---- GPU: rope ----------------------------------------------------------------------------------

def plain_rope(x, pos, rot, layout, freq, mscale):
    x = x.double().cpu().numpy()
    ang = pos[:, None].astype(np.float64) * freq[None]
    c, s = np.cos(ang)[:, None] * mscale, np.sin(ang)[:, None] * mscale
    i0 = np.arange(rot // 2) if layout == "half" else np.arange(0, rot, 2)
    i1 = i0 + rot // 2 if layout == "half" else i0 + 1
    y, mag = x.copy(), np.zeros_like(x)
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    mag[..., i0] = mag[..., i1] = (np.abs(x[..., i0]) + np.abs(x[..., i1])) * mscale
    return y, mag


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout,scaling", [("half", "none"), ("half", "yarn"), ("interleaved", "linear"),
                                            ("interleaved", "none")])
@pytest.mark.parametrize("n,hq,hk,d,rot,hi,how", [
    (1, 1, 0, 64, 64, 10, "new"), (64, 16, 2, 256, 64, 32768, "new"), (7, 3, 1, 128, 128, 1 << 20, "place"),
    (33, 4, 4, 64, 16, 2 ** 31 - 1, "strided"), (9, 5, 1, 72, 48, 4096, "odd"), (1000, 8, 2, 128, 32, 131072, "place")])
def test_rope(lib, dtype, layout, scaling, n, hq, hk, d, rot, hi, how):
    g = torch.Generator().manual_seed(n + rot)
    pos = np.random.default_rng(n).integers(0, hi, n).astype(np.int32)
    if n > 2:
        pos[0], pos[1], pos[2] = 0, hi - 1, -1
    wide = torch.randn(n, hq + hk + 1, d + 8, generator=g).to(DEV, dtype)
    if how == "strided":
        q, k = wide[:, :hq, :d], wide[:, hq:hq + hk, :d]
    elif how == "odd":  # not 16-byte aligned
        q, k = wide[:, :hq, 1:d + 1], wide[:, hq:hq + hk, 3:d + 3]
    else:
        q, k = wide[:, :hq, :d].contiguous(), wide[:, hq:hq + hk, :d].contiguous()
    plan = kv8.RopePlan(d, rot, theta=1e6, layout=layout, scaling=scaling, factor=4.0)
    freq, m = plain_freq(rot, 1e6, scaling, 4.0)
    q0, k0 = q.clone(), k.clone()
    if how == "place":
        yq, yk = kv8.rope(plan, q, k, dev32(pos), q_out=q, k_out=k)
    else:
        oq, ok = torch.full(q.shape, 5.0, dtype=dtype, device=DEV), torch.full(k.shape, 5.0, dtype=dtype, device=DEV)
        yq, yk = kv8.rope(plan, q, k if hk else None, dev32(pos), q_out=oq, k_out=ok if hk else None)
        assert torch.equal(q, q0)
    for x, y in ((q0, yq), (k0, yk)):
        if not x.shape[1]:
            continue
        want, mag = plain_rope(x, pos, rot, layout, freq, float(np.float32(m)))
        got = y.double().cpu().numpy()
        # sin and cos within 3 roundings (their own 2 and the factor's), two products and a sum;
        # the reduction of pos * f in 64 bits is off by 2^-52 of the angle
        tol = mag * (6 * F32_STEP + hi * 2.0 ** -51) + (np.abs(want) * BF16_STEP if dtype == torch.bfloat16 else 0)
        skip = pos < 0
        assert (np.abs(got - want)[~skip] <= tol[~skip] + 1e-30).all()
        np.testing.assert_array_equal(got[..., rot:][~skip], x.double().cpu().numpy()[..., rot:][~skip])
        kept = x.double().cpu().numpy()[skip] if how == "place" else 5.0
        assert (got[skip] == kept).all()


@pytest.mark.gpu
def test_rope_refusals(lib):
    plan = kv8.RopePlan(64)
    q, pos = torch.zeros(4, 2, 64, device=DEV), dev32([0, 1, 2, 3])
    for bad in (dict(q=q.half()), dict(q=q[:3]), dict(q=q[..., :32]), dict(positions=pos.long()),
                dict(k=q.bfloat16()), dict(q_out=q[:, :1])):
        with pytest.raises(DmError):
            kv8.rope(**{**dict(plan=plan, q=q, k=None, positions=pos), **bad})
    with pytest.raises(DmError):  # the same tensor under other strides
        kv8.rope(plan, q, None, pos, q_out=q.as_strided(q.shape, (64, 256, 1)))


# ---- GPU: append ----------------------------------------------------------------------------------

def slots_for(ctx, new, seed, spare=3):
    lens = [c + w for c, w in zip(ctx, new)]
    n_pages = sum(-(-n // PAGE) for n in lens) + spare
    table = make_table(lens, n_pages, seed)
    slots = [table[i, p // PAGE] * PAGE + p % PAGE for i in range(len(ctx)) for p in range(ctx[i], lens[i])]
    return n_pages, table, np.asarray(slots, np.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hk,d", [(1, 64), (2, 256), (3, 128)])
@pytest.mark.parametrize("ctx,new,how", [([0], [1], ""), ([5], [1], ""), ([15, 16, 17, 0], [1, 1, 1, 1], "pad"),
                                         ([3, 0, 31], [30, 16, 2], "strided"), ([0, 7], [700, 600], "odd"),
                                         ([4, 9, 14], [2, 3, 1], "grow"), ([2], [1600], "")])
def test_append(lib, dtype, hk, d, ctx, new, how):
    n_pages, _, slots = slots_for(ctx, new, len(ctx))
    cache = make_cache(n_pages, hk, d, 1, lo=-12, hi=0)
    g = torch.Generator().manual_seed(d)
    wide = torch.randn(len(slots), 2 * hk, d + 8, generator=g)
    wide *= torch.exp2(torch.randint(-9, 12 if how == "grow" else 2, (len(slots), 2 * hk, 1), generator=g))
    wide = wide.to(DEV, dtype)
    a = 1 if how == "odd" else 0
    k, v = wide[:, :hk, a:d + a], wide[:, hk:, a:d + a]
    if how not in ("strided", "odd"):
        k, v = k.contiguous(), v.contiguous()
    if how == "pad":
        slots = np.concatenate([slots, [-1, -1]]).astype(np.int32)
        k, v = (torch.cat([x, torch.full((2, hk, d), 1e30, dtype=dtype, device=DEV)]) for x in (k, v))
    p0, s0 = cache.pages.cpu().numpy().copy(), cache.scales.cpu().numpy().copy()
    err = kv8.error_word()
    kv8.append(cache, k, v, dev32(slots), err=err)
    kv8.check(err)
    pages, scales = plain_append(p0, s0, k.float().cpu().numpy(), v.float().cpu().numpy(), slots)
    np.testing.assert_array_equal(cache.scales.cpu().numpy(), scales.astype(np.float32))
    got = cache.pages.cpu().numpy()
    # the sign of a rounded-away negative value is kept by both
    np.testing.assert_array_equal(got, pages)


@pytest.mark.gpu
def test_append_extremes(lib):
    """Zeros, subnormals, values at the edge of a scale, the largest floats, Inf and NaN."""
    cache = kv8.Kv8Cache.empty(8, 1, 64)
    rows = [0.0, 2.0 ** -140, 448.0, 448.0 * (1 + 2.0 ** -20), 3.5, 3.4e38, 1e-38, 7.0]
    k = torch.tensor(rows)[:, None, None].expand(-1, 1, 64).clone()
    k[:, :, 1] *= -0.3
    v = k.clone()
    slots = np.arange(8, dtype=np.int32) * PAGE
    err = kv8.error_word()
    kv8.append(cache, k.to(DEV), v.to(DEV), dev32(slots), err=err)
    kv8.check(err)
    pages, scales = plain_append(np.zeros((8, 2, 1, 16, 64), np.uint8), np.full((8, 2, 1), 2.0 ** -100), k.numpy(),
                                 v.numpy(), slots)
    np.testing.assert_array_equal(cache.scales.cpu().numpy(), scales.astype(np.float32))
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), pages)
    k[1, 0, 3], k[2, 0, 4], k[2, 0, 5] = float("nan"), float("inf"), -float("inf")
    kv8.append(cache, k.to(DEV), v.to(DEV), dev32(slots), err=err)
    with pytest.raises(DmError) as e:
        kv8.check(err)
    assert e.value.code == _lib.DM_ERR_NONFINITE
    pages, scales = plain_append(pages, scales, k.numpy(), v.numpy(), slots)
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), pages)


@pytest.mark.gpu
def test_append_bad_slots(lib):
    """A slot behind the cache and rows out of order are left out and reported."""
    cache = kv8.Kv8Cache.empty(4, 1, 64)
    x = torch.randn(5, 1, 64, device=DEV)
    err = kv8.error_word()
    kv8.append(cache, x, x, dev32([64, 5, 2 ** 31 - 1, 30, -9]), err=err)
    with pytest.raises(DmError) as e:
        kv8.check(err)
    assert e.value.code == _lib.DM_ERR_INVALID_ARG
    touched = cache.pages.cpu().numpy().reshape(4, 2, 16, 64).any(axis=(1, 3))
    assert sorted(map(tuple, np.argwhere(touched))) == [(0, 5), (1, 14)]
    kv8.append(cache, x, x, dev32([32, 33, 35, 33, 34]), err=err)  # 35 breaks the order
    with pytest.raises(DmError):
        kv8.check(err)
    touched = cache.pages.cpu().numpy().reshape(4, 2, 16, 64).any(axis=(1, 3))
    assert touched[2, :2].all() and not touched[2, 2:].any()


# ---- GPU: attention ---------------------------------------------------------------------------------

SHAPES = [(1, 4, 64), (2, 8, 256), (2, 1, 128), (1, 16, 128), (2, 3, 64), (1, 6, 256), (1, 11, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hk,grp,d", SHAPES)
@pytest.mark.parametrize("lens", [[1], [0, 1, 15, 16, 17], [300, 0, 64, 65, 1000, 7, 33], [2111]])
def test_attention_one_token(lib, dtype, hk, grp, d, lens):
    check_attention(lens, [1] * len(lens), hk, grp, d, dtype, seed=len(lens), cu_none=len(lens) % 2 == 0,
                    extra=len(lens) % 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hk,grp,d", SHAPES)
@pytest.mark.parametrize("lens,rows", [([5, 40, 3], [2, 7, 3]), ([130, 0, 17], [130, 0, 1]), ([200, 90], [33, 64]),
                                       ([3, 2], [5, 2])])
def test_attention_chunks(lib, dtype, hk, grp, d, lens, rows):
    check_attention(lens, rows, hk, grp, d, dtype, seed=7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,len_hi,q_hi", [(65, 300, 1), (97, 500, 4), (70, 150, 40), (80, 40, 40), (600, 30, 1)])
def test_attention_many_requests(lib, dtype, n, len_hi, q_hi):
    """More than 64 requests, empty ones and ones without a query among them."""
    g = np.random.default_rng(n)
    lens, rows = g.integers(0, len_hi + 1, n), g.integers(0, q_hi + 1, n)
    rows = np.minimum(rows, np.maximum(lens, 1))
    check_attention([int(x) for x in lens], [int(x) for x in rows], 1, 8, 64, dtype, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grp,d,rows", [(16, 64, 1), (2, 64, 1), (9, 128, 1), (1, 256, 1), (8, 64, 4), (1, 128, 40)])
def test_attention_many_tiles(lib, dtype, grp, d, rows):
    """Enough keys that every CTA runs through its ring of tiles several times (148 SMs, two CTAs
    each, 12 tiles of 128 keys in a ring: 2 * 148 * 24 * 128 keys)."""
    n = 13
    lens = [2 * 148 * 24 * 128 // n + 37 * i for i in range(n)]
    check_attention(lens, [rows] * n, 1, grp, d, dtype, seed=8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_long_prompt(lib, dtype):
    check_attention([601, 300], [601, 129], 1, 2, 128, dtype, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_uneven_scales(lib, dtype, rows):
    """Page scales 2^40 apart, one peaked and one flat row, a large and a tiny softmax scale."""
    def spread(cache, table, q):
        g = np.random.default_rng(5)
        cache.scales[:, 1] = torch.from_numpy(np.exp2(g.integers(-30, 11, tuple(cache.scales[:, 1].shape))).astype(np.float32)).to(DEV)
        q[0] *= 20
        q[-1] *= 1e-6
    for scale in (None, 1e-4, -0.05):
        check_attention([700, 90], [rows, rows], 2, 4, 128, dtype, seed=2, scale=scale, mutate=spread)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 256])
def test_attention_nan_in_masked_places(lib, dtype, d):
    """NaN codes behind the last key and under the causal mask do not reach a query; a visible
    one does."""
    lens, rows = [37, 70, 20], [1, 50, 3]

    def poison(cache, table, q):
        for i, n in enumerate(lens):
            cache.pages[table[i, (n - 1) // PAGE], :, :, (n - 1) % PAGE + 1:] = 0x7f
    cache, table, cu, q, clean = check_attention(lens, rows, 2, 4, d, dtype, seed=4, mutate=poison)
    cache.pages[int(table[1, 40 // PAGE]), 1, 0, 40 % PAGE, 3] = 0xff  # request 1, V of key 40, kv head 0
    cache.pages[int(table[1, 60 // PAGE]), 0, 1, 60 % PAGE, 5] = 0x7f  # K of key 60, kv head 1
    got = kv8.attention(cache, q, dev32(table), dev32(lens), dev32(cu), 50,
                        workspace=kv8.attention_workspace(cache)).float().cpu().numpy()
    want = clean.float().cpu().numpy()
    pos = np.arange(50) + 20  # positions of request 1's queries
    for h in range(8):
        hit = pos >= (40 if h < 4 else 60)
        assert np.isnan(got[1:51, h][hit]).any(axis=-1).all()
        np.testing.assert_array_equal(got[1:51, h][~hit], want[1:51, h][~hit])
    np.testing.assert_array_equal(got[[0, 51, 52, 53]], want[[0, 51, 52, 53]])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_leaves_other_rows(lib, rows):
    """Rows behind the last request stay; a request with too many queries, a bad page and a
    length beyond the table are reported and touch nothing else."""
    lens = [60, 75]
    cache, table, cu, q, want = check_attention(lens, [rows, rows], 1, 4, 64, torch.bfloat16, seed=9)
    ws, err = kv8.attention_workspace(cache), kv8.error_word()
    pad = torch.cat([q, q])
    out = torch.full(pad.shape, 3.0, dtype=q.dtype, device=DEV)
    kv8.attention(cache, pad, dev32(table), dev32(lens), dev32(cu), rows, out=out, workspace=ws, err=err)
    kv8.check(err)
    assert torch.equal(out[:2 * rows], want) and (out[2 * rows:] == 3).all()
    # request 0 with more queries than max_q_len
    if rows > 1:
        out.fill_(3.0)
        kv8.attention(cache, q, dev32(table), dev32(lens), dev32([0, rows + 1, 2 * rows]), rows, out=out, workspace=ws,
                      err=err)
        with pytest.raises(DmError):
            kv8.check(err)
        assert (out[:rows + 1] == 3).all() and not (out[rows + 1:2 * rows] == 3).all(-1).any()  # every row written
    # a page out of range: its keys are left out (request 1's second page)
    bad = table.copy()
    bad[1, 1] = cache.num_pages
    got = kv8.attention(cache, q, dev32(bad), dev32(lens), dev32(cu), rows, workspace=ws, err=err)
    with pytest.raises(DmError):
        kv8.check(err)
    assert torch.equal(got[:rows], want[:rows]) and got.isfinite().all()
    # a length beyond the table's width
    got = kv8.attention(cache, q, dev32(table), dev32([60, 16 * table.shape[1] + 1]), dev32(cu), rows, workspace=ws,
                        err=err)
    with pytest.raises(DmError) as e:
        kv8.check(err)
    assert e.value.code == _lib.DM_ERR_CAPACITY and torch.equal(got[:rows], want[:rows])


@pytest.mark.gpu
def test_attention_device_refusals(lib):
    """Refused on the host: a workspace that is too small, host memory for the cache, tensors
    of the wrong type or shape."""
    cache = kv8.Kv8Cache.empty(4, 2, 64)
    q, t, n = torch.zeros(1, 4, 64, device=DEV), dev32([[0, 1]]), dev32([5])
    ws = kv8.attention_workspace(cache)
    kv8.attention(cache, q, t, n, workspace=ws)
    for bad in (dict(workspace=ws[:-256]), dict(q=q.half()), dict(q=q[..., :32]), dict(q=q[:, :3]),
                dict(block_table=t.long()), dict(seq_lens=n.cpu()), dict(out=q[:0]), dict(cu_q=n),
                dict(lse=torch.zeros(1, 3, device=DEV)), dict(max_q_len=2), dict(sm_scale=math.inf)):
        with pytest.raises(DmError):
            kv8.attention(**{**dict(cache=cache, q=q, block_table=t, seq_lens=n, workspace=ws), **bad})
    host = torch.zeros(4, 2, 2, 16, 64, dtype=torch.uint8).pin_memory()
    c = _lib.DmKv8Cache(host.data_ptr(), cache.scales.data_ptr(), 4, 2, 64, 0)
    x, s = torch.zeros(1, 2, 64, device=DEV), dev32([0])
    rc, err = _call(lib, "dm_kv8_append", C.addressof(c), 1, 1, x.data_ptr(), 128, 64, x.data_ptr(), 128, 64,
                    s.data_ptr(), None, None)
    assert rc == _lib.DM_ERR_INVALID_ARG and "device memory" in err["detail"]


@pytest.mark.gpu
def test_attention_strides_stream_and_repeats(lib):
    """Strided q and out, a stream of its own, the same workspace call after call: the same
    bits as the contiguous call."""
    lens, rows = [500, 1200, 3], [1, 1, 1]
    cache, table, cu, q, want = check_attention(lens, rows, 2, 4, 128, torch.float32, seed=12)
    wide = torch.zeros(3, 16, 136, device=DEV)
    wide[:, ::2, 4:132] = q
    out = torch.zeros(3, 9, 128, device=DEV)
    ws = kv8.attention_workspace(cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            kv8.attention(cache, wide[:, ::2, 4:132], dev32(table), dev32(lens), out=out[:, 1:], workspace=ws)
    side.synchronize()
    assert torch.equal(out[:, 1:], want) and (out[:, 0] == 0).all()


@pytest.mark.gpu
def test_two_graphs_share_a_workspace(lib):
    """Two captured calls of different shapes on one workspace, replayed in turn on another
    stream than they were captured on: the same bits as eager calls."""
    cache, table, cu, q, want = check_attention([900, 2500, 40], [1, 1, 1], 2, 8, 64, torch.bfloat16, seed=3)
    q2 = torch.randn(60, 16, 64, generator=torch.Generator().manual_seed(1)).to(DEV, torch.bfloat16)
    t, n1, n2, cu2 = dev32(table), dev32([900, 2500, 40]), dev32([700, 30, 33]), dev32([0, 20, 40, 60])
    ws = kv8.attention_workspace(cache)
    want2 = kv8.attention(cache, q2, t, n2, cu2, 20, workspace=ws)
    out, out2 = torch.empty_like(q), torch.empty_like(q2)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[0]):
        kv8.attention(cache, q, t, n1, out=out, workspace=ws)
    with torch.cuda.graph(graphs[1]):
        kv8.attention(cache, q2, t, n2, cu2, 20, out=out2, workspace=ws)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for i in range(6):
            out.zero_(), out2.zero_()
            graphs[i % 2].replay()
            graphs[(i + 1) % 2].replay()
            side.synchronize()
            assert torch.equal(out, want) and torch.equal(out2, want2)


@pytest.mark.gpu
def test_attention_repeats_bit_for_bit(lib):
    """Split requests are joined in a fixed order whatever the arrival order."""
    cache, table, cu, q, want = check_attention([30000, 5, 17001], [1, 1, 1], 2, 4, 128, torch.float32, seed=6)
    ws = kv8.attention_workspace(cache)
    for _ in range(20):
        assert torch.equal(kv8.attention(cache, q, dev32(table), dev32([30000, 5, 17001]), workspace=ws), want)


@pytest.mark.gpu
def test_outputs_follow_the_given_stream(lib):
    """Outputs that a call with `stream` allocates belong to that stream: memory that the current
    stream still uses is not handed out."""
    side = torch.cuda.Stream()
    plan, pos = kv8.RopePlan(64), dev32(range(512))
    q = torch.randn(512, 8, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    want, _ = kv8.rope(plan, q, None, pos)
    torch.cuda.synchronize()
    for s in (side.cuda_stream, 0):
        busy = torch.empty_like(q)
        for _ in range(50):
            busy.fill_(1.0)
        del busy  # its memory is free for the current stream alone
        got, _ = kv8.rope(plan, q, None, pos, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_gradients_are_refused(lib):
    cache = kv8.Kv8Cache.empty(4, 2, 64)
    q = torch.zeros(1, 4, 64, device=DEV, requires_grad=True)
    k = torch.zeros(1, 2, 64, device=DEV)
    ws, one = kv8.attention_workspace(cache), dev32([1])
    for call in (lambda: kv8.rope(kv8.RopePlan(64), q, None, one),
                 lambda: kv8.append(cache, k, q[:, :2], dev32([0])),
                 lambda: kv8.attention(cache, q, dev32([[0]]), one, workspace=ws)):
        with pytest.raises(DmError, match="gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", ["kv8_append", "kv8_attn", "kv8_plan", "kv8_rope"])
@pytest.mark.parametrize("batch,ctx,new", [(2, 100, 1), (3, 70, 33), (1, 16, 16)])
def test_kernel_bench_runs(lib, capsys, monkeypatch, kernel, batch, ctx, new):
    from disk_streaming_moe_engine_b200 import kernel_bench
    monkeypatch.setattr("sys.argv", ["kernel_bench", "--preset", "mini", "--kernel", kernel, "--batch", str(batch),
                                     "--ctx", str(ctx), "--new", str(new), "--iters", "2"])
    kernel_bench.main()
    line = json.loads(capsys.readouterr().out)
    assert line["kernel"] == kernel and line["us"] > 0 and line["bytes"] > 0


# ---- GPU: the chain as a server runs it ---------------------------------------------------------------

@pytest.mark.gpu
def test_serving_chain_and_captured_step(lib):
    """Prompts, then decode steps through a captured graph with one request ending: the
    attention over what the chain stored equals 64-bit attention over the stored values, which
    are the plain append of the rotated keys; the pages return to the free list."""
    hk, grp, d, n, cap, width = 2, 4, 64, 5, 40, 8
    g = torch.Generator().manual_seed(0)
    cache = kv8.Kv8Cache.empty(cap, hk, d)
    free, state = kv8.free_list(cap)
    table = torch.zeros((n, width), dtype=torch.int32, device=DEV)
    lens = torch.zeros(n, dtype=torch.int32, device=DEV)
    rp = kv8.RopePlan(d, 32, theta=1e6, layout="interleaved", scaling="yarn", factor=4.0)
    ws, err = kv8.attention_workspace(cache), kv8.error_word()
    new = [33, 1, 16, 50, 7]
    tokens = sum(new)

    def step(q, k, v, new_t, max_tokens, max_q, out):
        plan = kv8.plan_slots(free, state, table, lens, new_t, max_tokens, out=out, err=err)
        q, k = kv8.rope(rp, q, k, plan.positions, q_out=q, k_out=k)
        kv8.append(cache, k, v, plan.slots, err=err)
        return kv8.attention(cache, q, table, plan.seq_lens, plan.cu_new, max_q, workspace=ws, err=err)

    def outputs(max_tokens):
        z = torch.zeros((3, max_tokens), dtype=torch.int32, device=DEV)
        return kv8.SlotPlan(lens, torch.zeros(n + 1, dtype=torch.int32, device=DEV), z[0], z[1], z[2])

    def check_step(q, plan, got, rows):
        kv8.check(err)
        ll, cu = lens.cpu().numpy(), plan.cu_new.cpu().numpy()
        np.testing.assert_array_equal(np.diff(cu), rows)
        out, mag, sat, _ = plain_attention(cache, q, table.cpu().numpy(), ll, cu, d ** -0.5)
        live = int(cu[-1])
        diff = np.abs(got.double().cpu().numpy()[:live] - out[:live])
        assert (diff <= attention_tolerance(out, mag, sat, d, ll.max(), q.dtype)[:live]).all()

    q, k, v = (torch.randn(tokens, h, d, generator=g).to(DEV) for h in (hk * grp, hk, hk))
    prompt = outputs(tokens)
    empty = cache.pages.cpu().numpy().copy(), cache.scales.cpu().numpy().copy()
    got = step(q, k, v, dev32(new), tokens, 50, prompt)
    check_step(q, prompt, got, new)
    pages, scales = plain_append(*empty, k.cpu().numpy(), v.cpu().numpy(), prompt.slots.cpu().numpy())
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), pages)
    # decode steps in a graph: fixed buffers, a padded token row, lengths in place
    q, k, v = (torch.zeros(n, h, d, device=DEV) for h in (hk * grp, hk, hk))
    new_t, decode = dev32([1] * n), outputs(n)
    out = torch.zeros(n, hk * grp, d, device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out.copy_(step(q, k, v, new_t, n, 1, decode))
    for s in range(20):
        rows = [1] * n
        if s >= 10:
            rows[3] = -1 if s == 10 else 0
        new_t.copy_(dev32(rows))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        graph.replay()
        check_step(q, decode, out, [max(r, 0) for r in rows])
    assert lens.tolist() == [53, 21, 36, 0, 27]
    held = sum(-(-x // PAGE) for x in lens.tolist())
    assert state.tolist() == [cap - held, 0]
    used = [int(table[i, p]) for i in range(n) for p in range(-(-int(lens[i]) // PAGE))]
    assert sorted(used + free[:cap - held].tolist()) == list(range(cap))
