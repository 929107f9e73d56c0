"""The 8-bit cache operators at the ends of what their contract allows: softmax weights far below
the largest, page scales far apart, queries of extreme size, codes that are NaN, rows that no
request covers, calls from several threads."""
import math
import threading

import numpy as np
import pytest
import torch

from disk_streaming_moe_engine_b200 import DmError, _lib, kv8
from test_kv8 import BF16_STEP, DEV, E4M3, PAGE, dev32, make_cache, make_table, plain_attention

F16_STEP = 2.0 ** -11  # largest relative rounding of fp16


def query_side(n, max_q, group, hk, dtype):
    """The rule between the two attention kernels: True where 128 query rows go on the M side."""
    rows = max_q * group
    items = -(-rows // 128) * n * hk
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return dtype == torch.bfloat16 and rows >= (40 if 2 * items >= sms else 96 if items >= 8 else 192)


def tolerance(cache, q, scale, ref, keys, on_query_side):
    """Per output.  A score's error e changes an output by at most 2 e sum p |v|.  e: products and
    sums in fp32 (D / 16 + 1 chained sums, 2^-22 of the magnitudes each), and q as e4m3 terms: bf16
    on the query side off by 2^-17 of the row's largest element, on the key side by 2^-21 of it;
    fp32 by 2^-20 of the element or 2^-26 of 2^8, the largest being at least 2^7.  Weights, sums in
    fp32: on the query side three e5m2 terms of 2^11 w, each holding the next 3 bits: off by 2^-9 of
    themselves (and 2^-11 on the way through fp16) or 2^-28 (half of 2^-16 / 2^11).  On the key side e4m3 terms of 64 w, or of 2^20 w for w < 2^-12, each term off by 2^-4 of
    itself and the next one holding 16 times that: three terms 2^-12 (and 2^-11 on the way through
    fp16) or 2^-38 (half of 2^-9 / 256 / 2^20), five 2^-20 or 2^-46.  What is absolute is relative to
    a reference that the row's largest p sV is never below; doubled or
    more for the rounding on the way.  bf16 results are rounded once."""
    out, (mag, small), sat, _ = ref
    d, bf16 = q.shape[-1], q.dtype == torch.bfloat16
    k = torch.from_numpy(E4M3).to(DEV)[cache.pages[:, 0].long()].nan_to_num() * cache.scales[:, 0, :, None, None].double()
    size = (q.double().abs().amax(-1) * k.abs().sum(-1).max() * abs(scale)).cpu().numpy()
    e = sat * (d / 16 + 1) * 2.0 ** -22 + size * ((2.0 ** -17 if on_query_side else 2.0 ** -21) if bf16 else 2.0 ** -25)
    if not bf16:
        e = e + sat * 2.0 ** -20
    rel, low = (2.0 ** -9 + F16_STEP, 2.0 ** -27) if on_query_side else (2.0 ** -12 + F16_STEP, 2.0 ** -36) if bf16 else (2.0 ** -20, 2.0 ** -44)
    tol = (2 * e[..., None] + (keys / PAGE + 4) * 2.0 ** -22 + rel) * mag + low * small
    return tol + (BF16_STEP * np.abs(out) if bf16 else 0) + 1e-30, e


def check_against_64_bits(cache, q, table, lens, rows, scale, max_q=None):
    """attention() over all rows against the plain form; (results, lse, reference)."""
    cu = np.concatenate([[0], np.cumsum(rows)])
    max_q = max_q or max(rows)
    err = kv8.error_word()
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = kv8.attention(cache, q, dev32(table), dev32(lens), dev32(cu), max_q, sm_scale=scale, lse=lse,
                        workspace=kv8.attention_workspace(cache), err=err)
    kv8.check(err)
    ref = plain_attention(cache, q, table, lens, cu, scale)
    side = query_side(len(lens), max_q, q.shape[1] // cache.num_kv_heads, cache.num_kv_heads, q.dtype)
    tol, e = tolerance(cache, q, scale, ref, max(lens), side)
    diff = np.abs(got.double().cpu().numpy() - ref[0])
    assert (diff <= tol).all(), (np.nanmax(diff / tol), np.isnan(diff).any())
    want = ref[3]
    at = np.isfinite(want)
    sums = lse.double().cpu().numpy()
    assert (np.isneginf(sums) == ~at).all()
    assert (np.abs(sums[at] - want[at]) <= e[at] + np.abs(want[at]) * 2.0 ** -22 + 2.0 ** -18).all()
    return got, lse, ref


# ---- softmax weights far below the largest ------------------------------------------------------------

def peaked(d, hk, grp, keys, rows, nats, at, seed):
    """One key whose score is `nats` above the others' mean (their spread about 1/2), with V = 0
    there: the result is the other keys' alone, whose weights are e^-nats and less."""
    g = torch.Generator().manual_seed(seed)
    cache = make_cache(-(-keys // PAGE) + 2, hk, d, seed)
    u = torch.randint(0, 2, (d,), generator=g) * 2.0 - 1
    c = nats / (2 * math.sqrt(d))
    tail = (torch.randn(cache.num_pages, hk, PAGE, d, generator=g) * (math.sqrt(d) / nats)).to(torch.float8_e4m3fn)
    cache.pages[:, 0] = tail.view(torch.uint8).to(DEV)
    cache.scales[:, 0] = 1.0
    cache.scales[:, 1] = 2.0 ** -7
    table = make_table([keys], cache.num_pages, seed)
    page, off = int(table[0, at // PAGE]), at % PAGE
    cache.pages[page, 0, :, off] = (2 * u).to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
    cache.pages[page, 1, :, off] = 0
    q = u * c * (1 + 0.05 * torch.rand(rows, hk * grp, 1, generator=g)) + 0.01 * torch.randn(rows, hk * grp, d, generator=g)
    return cache, table, q


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,grp", [(1, 8), (1, 11), (48, 4)])
@pytest.mark.parametrize("keys,nats,at", [(8192, 11, 0), (8192, 14, 4000), (32768, 12, 5), (8192, 19, 8100), (130, 14, 64)])
def test_small_weights_count(lib, dtype, d, rows, grp, keys, nats, at):
    """The key side (one token) and the query side (48 tokens of 4 heads, bf16): thousands of keys
    11 to 19 nats below one that adds nothing, or a few in its own tile."""
    cache, table, q = peaked(d, 1, grp, keys, rows, nats, at, seed=keys + nats)
    q = q.to(DEV, dtype)
    assert query_side(1, rows, grp, 1, dtype) == (rows == 48 and dtype == torch.bfloat16)
    got, _, ref = check_against_64_bits(cache, q, table, [keys], [rows], d ** -0.5)
    assert np.abs(ref[0]).max() > 0 and (got != 0).any()


# ---- V page scales far apart ------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,grp", [(1, 2), (48, 4)])
@pytest.mark.parametrize("high,low,how", [(27, -100, "alternate"), (100, -100, "alternate"), (100, -100, "low first"),
                                          (100, -100, "high first"), (0, -100, "low first"), (60, -60, "alternate"),
                                          (-95, -100, "alternate")])
def test_v_scales_far_apart(lib, dtype, rows, grp, high, low, how):
    """A key's share of the softmax does not depend on its V: pages of all-zero V (scale 2^-100)
    beside pages of huge V, in one tile and in different ones, in one CTA and in several."""
    d, keys = 64, 3000
    cache = make_cache(-(-keys // PAGE) + 1, 1, d, seed=3, lo=-8, hi=-8)
    table = make_table([keys], cache.num_pages, 3)
    n = table.shape[1]
    is_low = {"alternate": np.arange(n) % 2 == 1, "low first": np.arange(n) < n // 2,
              "high first": np.arange(n) >= n // 2}[how]
    for page, lo in zip(table[0], is_low):
        cache.scales[page, 1] = 2.0 ** (low if lo else high)
        if lo and low == -100:
            cache.pages[page, 1] = 0
    q = torch.randn(rows, grp, d, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
    check_against_64_bits(cache, q, table, [keys], [rows], d ** -0.5)
    check_against_64_bits(cache, q, table[:, :8], [100], [rows], d ** -0.5)


# ---- calls from several threads --------------------------------------------------------------------------

@pytest.mark.gpu
def test_plans_of_different_sizes_from_several_threads(lib):
    """The plan of many requests needs more shared memory than that of fewer: a call on another
    thread does not take it away between the setting and the launch."""
    import ctypes as C
    failed = []

    def work(n, stream):
        ctx, new = dev32([0] * n), dev32([1] * n)
        table = torch.zeros((n, 1), dtype=torch.int32, device=DEV)
        free, state = kv8.free_list(n)
        left, tok = dev32([0, 0]), torch.zeros((4, n + 1), dtype=torch.int32, device=DEV)
        lens, buf = torch.zeros_like(ctx), C.create_string_buffer(512)
        ptr = [C.c_void_p(t.data_ptr()) for t in (ctx, new, table, free, state, left, lens, *tok)]
        args = (n, *ptr[:3], 1, ptr[3], n, *ptr[4:7], ptr[7], n, *ptr[8:], None, C.c_void_p(stream.cuda_stream), buf, 512)
        torch.cuda.synchronize()
        for _ in range(10000):
            if lib.dm_kv8_plan(*args):
                failed.append((n, buf.value.decode()))
                break

    streams = [torch.cuda.Stream() for _ in range(6)]
    threads = [threading.Thread(target=work, args=a) for a in zip((8192, 3500, 8000, 3600, 8100, 4000), streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed


# ---- many short items ------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("empty", [0, 3, 40])
def test_many_short_items_on_the_query_side(lib, empty):
    """Items of one tile, requests without tokens between them: every warp of a CTA walks over many
    items, and none may fall behind for good (the kernel's waits would run out)."""
    hk, grp, d, n = 2, 8, 64, 400
    lens = [0 if i % (empty + 1) else 60 for i in range(n)]
    rows = [0 if i % (empty + 1) else 9 + i % 12 for i in range(n)]
    cache = make_cache(n * 4 + 1, hk, d, 2)
    table = make_table(lens, cache.num_pages, 2)
    assert query_side(n, max(rows), grp, hk, torch.bfloat16)
    q = torch.randn(sum(rows), hk * grp, d, generator=torch.Generator().manual_seed(4)).to(DEV, torch.bfloat16)
    got, _, _ = check_against_64_bits(cache, q, table, lens, rows, d ** -0.5)
    cu, err, ws = dev32(np.concatenate([[0], np.cumsum(rows)])), kv8.error_word(), kv8.attention_workspace(cache)
    for _ in range(50):
        again = kv8.attention(cache, q, dev32(table), dev32(lens), cu, max(rows), workspace=ws, err=err)
        assert torch.equal(again, got)
    kv8.check(err)


# ---- what the operators refuse -----------------------------------------------------------------------------

@pytest.mark.gpu
def test_forward_mode_is_refused(lib):
    """A dual tensor's tangent would be lost without a word."""
    from torch.autograd import forward_ad
    cache = kv8.Kv8Cache.empty(4, 2, 64)
    x, one = torch.zeros(1, 2, 64, device=DEV), dev32([1])
    ws = kv8.attention_workspace(cache)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda t: kv8.rope(kv8.RopePlan(64), t, None, one),
                     lambda t: kv8.append(cache, x, t, dev32([0])),
                     lambda t: kv8.attention(cache, t, dev32([[0]]), one, workspace=ws)):
            call(x)
            with pytest.raises(DmError, match="gradient"):
                call(dual)


# ---- queries of extreme size -----------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,grp", [(2, 4), (48, 4)])
@pytest.mark.parametrize("power", [-112, -100, 0, 100, 112, 120])
def test_q_of_extreme_size(lib, dtype, rows, grp, power):
    """q times 2^power against keys times 2^-power (as far as the scales go, the softmax scale takes
    the rest): ordinary scores."""
    d, keys, k_power = 64, 500, max(-100, min(92, -power))
    cache = make_cache(-(-keys // PAGE) + 1, 1, d, 8, lo=-8, hi=-8)
    cache.scales[:, 0] = 2.0 ** (k_power - 8 if k_power > -92 else k_power)
    q = torch.randn(rows, grp, d, generator=torch.Generator().manual_seed(3)).clamp_(-4, 4)
    q = (q.double() * 2.0 ** power).to(DEV, dtype)
    rest = power + math.log2(float(cache.scales[0, 0, 0]))
    scale = d ** -0.5 * 2.0 ** (-rest - 8)
    check_against_64_bits(cache, q, make_table([keys], cache.num_pages, 8), [keys], [rows], scale)


# ---- rows that no request covers ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,grp", [(torch.float32, 5, 4), (torch.bfloat16, 5, 4), (torch.bfloat16, 60, 8)])
def test_allocated_outputs_have_no_stale_rows(lib, dtype, rows, grp):
    """attention() without `out`: rows that belong to no request, or to one that is skipped, are
    zeros, not what the memory held before."""
    lens, d = [70, 90, 40], 64
    cache = make_cache(20, 1, d, 1)
    table, ws = make_table(lens, 20, 1), kv8.attention_workspace(cache)
    total = 3 * rows + 7
    q = torch.randn(total, grp, d, generator=torch.Generator().manual_seed(0)).to(DEV, dtype)

    def written(got, a, b, length):
        """Rows a to b of a request: those that see a key have results, the others zeros."""
        sees = torch.arange(a, b, device=DEV) >= b - length
        return bool(((got[a:b] != 0).any(-1) == sees[:, None]).all())

    def run(cu, lengths, max_q=rows, rest=None):
        err = kv8.error_word()
        torch.cuda.synchronize()
        stale = [torch.full_like(q, math.nan) for _ in range(4)]
        del stale
        got = kv8.attention(cache, q, dev32(table), dev32(lengths), None if cu is None else dev32(cu), max_q,
                            workspace=ws, err=err)
        if rest is None:
            kv8.check(err)
        else:
            with pytest.raises(DmError):
                kv8.check(err)
        return got

    got = run([2, 2 + rows, 2 + 2 * rows, 3 * rows], lens)
    assert (got[:2] == 0).all() and (got[3 * rows:] == 0).all() and got[2:3 * rows].isfinite().all()
    assert written(got, 2, 2 + rows, 70) and written(got, 2 + rows, 2 + 2 * rows, 90) and written(got, 2 + 2 * rows, 3 * rows, 40)
    # request 1 has more rows than max_q_len
    got = run([0, 2, 2 + rows + 1, 2 * rows], lens, rest=True)
    assert (got[2:3 + rows] == 0).all() and (got[2 * rows:] == 0).all()
    assert written(got, 0, 2, 70) and written(got, 3 + rows, 2 * rows, 40)
    # row ranges outside q and backwards
    got = run([0, 3, 2, total + 5], lens, rest=True)
    assert (got[:2] != 0).any(-1).all() and (got[3:] == 0).all() and got.isfinite().all()
    if rows == 5:  # one row per request, more rows than requests
        got = run(None, lens, max_q=1)
        assert (got[3:] == 0).all() and (got[:3] != 0).any(-1).all()
        assert (run([0, 0, 0, 0], lens) == 0).all()


@pytest.mark.gpu
def test_errors_without_a_word_are_kept(lib):
    """Without `err` the device's own error word takes what only the device can see: a refused plan,
    a slot behind the cache and a request with too many rows raise at the next check()."""
    kv8.check()
    cache = kv8.Kv8Cache.empty(4, 1, 64)
    x, ws = torch.randn(3, 1, 64, device=DEV), kv8.attention_workspace(cache)
    free, state = kv8.free_list(1)
    kv8.plan_slots(free, state, torch.zeros((1, 4), dtype=torch.int32, device=DEV), dev32([0]), dev32([40]), 64)
    with pytest.raises(DmError) as e:
        kv8.check()
    assert e.value.code == _lib.DM_ERR_CAPACITY
    kv8.check()
    kv8.append(cache, x, x, dev32([0, 1, 4000]))
    with pytest.raises(DmError):
        kv8.check()
    kv8.attention(cache, x, dev32([[0]]), dev32([2]), dev32([0, 3]), 2, workspace=ws)
    with pytest.raises(DmError):
        kv8.check(device=x.device)
    kv8.check()
    graph, word, out = torch.cuda.CUDAGraph(), kv8.error_word(), torch.empty_like(x)
    args = (cache, x, dev32([[0]]), dev32([2]), dev32([0, 3]), 2)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kv8.attention(*args, out=out, workspace=ws)
    kv8.check()
    graph.replay()
    kv8.check(word)  # a word of one's own stays clean
    with pytest.raises(DmError):
        kv8.check()


@pytest.mark.gpu
def test_first_call_of_a_process_may_be_captured(lib):
    """Nothing that a call needs is made in a way that a capture forbids."""
    import subprocess
    import sys
    code = """
import torch
from disk_streaming_moe_engine_b200 import DmError, kv8
free, state = kv8.free_list(1)
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
table, ctx, new = torch.zeros((1, 4), dtype=torch.int32, device="cuda"), ints(0), ints(40)
tok = torch.zeros((5, 64), dtype=torch.int32, device="cuda")
out, graph = kv8.SlotPlan(*tok), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    kv8.plan_slots(free, state, table, ctx, new, 64, out=out)
graph.replay()
try:
    kv8.check()
except DmError as e:
    print("refused", e.code)
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert out.stdout.strip() == f"refused {_lib.DM_ERR_CAPACITY}", out.stderr[-2000:]


# ---- NaN codes of V ------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("keys,rows,grp,at", [(70, 50, 4, 40), (700, 60, 4, 655), (4000, 48, 4, 3960), (300, 1, 8, 299),
                                              (9000, 60, 4, 8990), (300, 20, 4, 10)])
def test_nan_of_v_reaches_its_element_alone(lib, dtype, d, keys, rows, grp, at):
    """softmax(q K^T) V with one NaN in V: every row that sees the key has that element NaN and no
    other, its lse is untouched; rows that do not see it are untouched."""
    cache = make_cache(-(-keys // PAGE) + 2, 2, d, 5)
    table = make_table([keys], cache.num_pages, 5)
    q = torch.randn(rows, 2 * grp, d, generator=torch.Generator().manual_seed(2)).to(DEV, dtype)
    ws, cu = kv8.attention_workspace(cache), [0, rows]

    def run():
        lse = torch.empty(q.shape[:2], device=DEV)
        got = kv8.attention(cache, q, dev32(table), dev32([keys]), dev32(cu), rows, workspace=ws, lse=lse,
                            out=torch.zeros_like(q))
        return got.float().cpu().numpy(), lse.cpu().numpy()
    want, want_lse = run()
    page = int(table[0, at // PAGE])
    cache.pages[page, 1, 0, at % PAGE, 3] = 0xff
    cache.pages[page, 1, 1, at % PAGE, d - 2] = 0x7f
    if at + 1 < keys:
        cache.pages[int(table[0, (at + 1) // PAGE]), 1, 1, (at + 1) % PAGE, d // 2] = 0x7f
    got, lse = run()
    np.testing.assert_array_equal(lse, want_lse)
    pos = np.arange(rows) + keys - rows
    nan = np.zeros(got.shape, bool)
    nan[pos >= at, :grp, 3] = True
    nan[pos >= at, grp:, d - 2] = True
    if at + 1 < keys:
        nan[pos >= at + 1, grp:, d // 2] = True
    assert (np.isnan(got) == nan).all()
    np.testing.assert_array_equal(got[~nan], want[~nan])


# ---- the query side at the sizes that the key side is tested at ------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("d,keys", [(64, 60000), (128, 50000), (256, 30000)])
def test_query_side_many_tiles(lib, d, keys):
    """Every CTA passes through its ring of slots and scales several times, items are joined from
    many parts."""
    lens, rows, grp = [keys, keys - 777, 40], [48, 50, 48], 4
    assert query_side(3, 50, grp, 1, torch.bfloat16)
    cache = make_cache(sum(-(-n // PAGE) for n in lens) + 1, 1, d, 4)
    table = make_table(lens, cache.num_pages, 4)
    q = torch.randn(sum(rows), grp, d, generator=torch.Generator().manual_seed(5)).to(DEV, torch.bfloat16)
    check_against_64_bits(cache, q, table, lens, rows, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("d,n,q_hi,grp", [(64, 66, 140, 8), (128, 70, 90, 12)])
def test_query_side_many_requests_of_many_rows(lib, d, n, q_hi, grp):
    """More than 64 requests of more than 1024 rows per kv head: blocks in pairs, not by exact tiles."""
    g = np.random.default_rng(n)
    rows = g.integers(0, q_hi + 1, n)
    rows[3] = q_hi
    lens = rows + g.integers(0, 200, n) * (g.random(n) < 0.7)
    assert q_hi * grp > 1024 and query_side(n, q_hi, grp, 1, torch.bfloat16)
    lens, rows = [int(x) for x in lens], [int(x) for x in rows]
    cache = make_cache(sum(-(-x // PAGE) for x in lens) + 1, 1, d, 6)
    table = make_table(lens, cache.num_pages, 6)
    q = torch.randn(sum(rows), grp, d, generator=torch.Generator().manual_seed(6)).to(DEV, torch.bfloat16)
    check_against_64_bits(cache, q, table, lens, rows, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 256])
def test_prompt_beside_single_tokens(lib, dtype, d):
    """A server's step: one prompt and one chunk among requests with a token each, in one call."""
    lens, rows, grp = [900] + [37 * i + 1 for i in range(40)] + [2000], [900] + [1] * 40 + [130], 4
    assert query_side(42, 900, grp, 2, dtype) == (dtype == torch.bfloat16)
    cache = make_cache(sum(-(-x // PAGE) for x in lens) + 1, 2, d, 7)
    table = make_table(lens, cache.num_pages, 7)
    q = torch.randn(sum(rows), 2 * grp, d, generator=torch.Generator().manual_seed(7)).to(DEV, dtype)
    check_against_64_bits(cache, q, table, lens, rows, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["strided", "odd"])
def test_query_side_strides(lib, how):
    """q and out as parts of larger tensors, at 32-byte boundaries and off them: the bits of the
    contiguous call, and nothing beside them is touched."""
    lens, rows, grp, d = [700, 333], [60, 50], 4, 128
    assert query_side(2, 60, grp, 2, torch.bfloat16)
    cache = make_cache(70, 2, d, 8)
    table = make_table(lens, 70, 8)
    q = torch.randn(110, 2 * grp, d, generator=torch.Generator().manual_seed(8)).to(DEV, torch.bfloat16)
    want, _, _ = check_against_64_bits(cache, q, table, lens, rows, d ** -0.5)
    a, pad = (16, 32) if how == "strided" else (1, 7)
    wide = torch.full((110, 2 * grp + 1, d + pad), 9.0, device=DEV, dtype=torch.bfloat16)
    out = torch.full((110, 3 * grp, d + pad), 5.0, device=DEV, dtype=torch.bfloat16)
    wide[:, 1:, a:a + d] = q
    kv8.attention(cache, wide[:, 1:, a:a + d], dev32(table), dev32(lens), dev32([0, 60, 110]), 60,
                  out=out[:, grp:, a:a + d], workspace=kv8.attention_workspace(cache))
    assert torch.equal(out[:, grp:, a:a + d], want)
    out[:, grp:, a:a + d] = 5.0
    assert (out == 5).all()


@pytest.mark.gpu
def test_query_side_leaves_other_rows(lib):
    """Rows behind the last request stay; a request with too many queries, a bad page and a length
    beyond the table are reported and touch nothing else."""
    lens, rows, grp, d = [260, 275], 100, 4, 64
    assert query_side(2, rows, grp, 1, torch.bfloat16)
    cache = make_cache(40, 1, d, 9)
    table = make_table(lens, 40, 9)
    q = torch.randn(2 * rows, grp, d, generator=torch.Generator().manual_seed(9)).to(DEV, torch.bfloat16)
    want, _, _ = check_against_64_bits(cache, q, table, lens, [rows, rows], d ** -0.5)
    ws, err, cu = kv8.attention_workspace(cache), kv8.error_word(), dev32([0, rows, 2 * rows])
    pad = torch.cat([q, q])
    out = torch.full(pad.shape, 3.0, dtype=q.dtype, device=DEV)
    kv8.attention(cache, pad, dev32(table), dev32(lens), cu, rows, out=out, workspace=ws, err=err)
    kv8.check(err)
    assert torch.equal(out[:2 * rows], want) and (out[2 * rows:] == 3).all()
    out.fill_(3.0)
    kv8.attention(cache, q, dev32(table), dev32(lens), dev32([0, rows + 1, 2 * rows]), rows, out=out, workspace=ws, err=err)
    with pytest.raises(DmError):
        kv8.check(err)
    assert (out[:rows + 1] == 3).all() and not (out[rows + 1:2 * rows] == 3).all(-1).any()
    bad = table.copy()
    bad[1, 1] = cache.num_pages
    got = kv8.attention(cache, q, dev32(bad), dev32(lens), cu, rows, workspace=ws, err=err)
    with pytest.raises(DmError):
        kv8.check(err)
    assert torch.equal(got[:rows], want[:rows]) and got.isfinite().all()
    got = kv8.attention(cache, q, dev32(table), dev32([260, 16 * table.shape[1] + 1]), cu, rows, workspace=ws, err=err)
    with pytest.raises(DmError) as e:
        kv8.check(err)
    assert e.value.code == _lib.DM_ERR_CAPACITY and torch.equal(got[:rows], want[:rows])


@pytest.mark.gpu
def test_calls_at_the_same_time(lib):
    """Both kernels on two streams at once, a workspace each, eager and as captured graphs: the bits
    of the calls alone."""
    d, grp = 128, 4
    cache = make_cache(900, 2, d, 10)
    cases = []
    for lens, rows, dtype in (([5000, 3000, 400], [1, 1, 1], torch.float32), ([2000, 900], [300, 64], torch.bfloat16)):
        table = make_table(lens, 900, len(lens))
        q = torch.randn(sum(rows), 2 * grp, d, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
        want, _, _ = check_against_64_bits(cache, q, table, lens, rows, d ** -0.5)
        args = (cache, q, dev32(table), dev32(lens), dev32(np.concatenate([[0], np.cumsum(rows)])), max(rows))
        cases.append((args, want, torch.cuda.Stream(), kv8.attention_workspace(cache), torch.zeros_like(q), torch.cuda.CUDAGraph()))
    torch.cuda.synchronize()
    for args, _, stream, ws, out, graph in cases:
        with torch.cuda.graph(graph, stream=stream):
            kv8.attention(*args, out=out, workspace=ws)
    err = kv8.error_word()
    for i in range(20):
        for args, _, stream, ws, out, graph in cases:
            with torch.cuda.stream(stream):
                out.zero_()
                if i % 2:
                    graph.replay()
                else:
                    kv8.attention(*args, out=out, workspace=ws, err=err)
        torch.cuda.synchronize()
        for _, want, _, _, out, _ in cases:
            assert torch.equal(out, want)
    kv8.check(err)


# ---- CPU: flags, and the arithmetic of the weights' terms --------------------------------------------------------

def test_attention_flags(lib):
    """DM_KV8_FILL_ROWS alone is known; an empty call needs no device."""
    import ctypes as C
    cache = _lib.DmKv8Cache(1 << 20, 1 << 21, 4, 2, 128, 0)
    for flags, want in ((0, _lib.DM_OK), (kv8.FILL_ROWS, _lib.DM_OK), (4, _lib.DM_ERR_INVALID_ARG), (3, _lib.DM_ERR_INVALID_ARG)):
        a = _lib.DmKv8AttnArgs(dtype=0, n=0, num_q_heads=8, max_q_len=1, rows=0, table_width=1, sm_scale=1.0, flags=flags)
        buf = C.create_string_buffer(512)
        assert lib.dm_kv8_attention(C.addressof(cache), C.addressof(a), None, buf, 512) == want


def test_three_e5m2_terms_hold_nine_bits():
    """Upper bytes of fp16 values: the value's, of what is left, of what is left then (rounded)."""
    x = np.exp2(np.random.default_rng(0).uniform(-30, 15, 200000))
    h = x.astype(np.float16)
    total = np.zeros_like(x)
    for i in range(3):
        bits = h.view(np.uint16)
        top = ((bits + 0x80) if i == 2 else bits) & 0xff00
        part = top.astype(np.uint16).view(np.float16)
        total += part.astype(np.float64)
        h = (h - part).astype(np.float16)
    off = np.abs(total - x)
    # the rounding to fp16 (2^-11, or half of its smallest step 2^-24) comes on top of what the terms
    # leave (2^-9, or half of e5m2's smallest step 2^-16)
    assert (off <= x * F16_STEP + 2.0 ** -25 + np.maximum(x * 2.0 ** -9, 2.0 ** -17)).all()
    assert total[x < 2.0 ** -26].max() == 0  # where a page's scores go that only count in the sum


def test_e4m3_terms_in_two_groups():
    """64 w, or 2^20 w below 2^-12, as three e4m3 terms of scales 1, 1/16, 1/256."""
    from test_kv8 import to_e4m3
    w = np.exp2(np.random.default_rng(1).uniform(-40, 2, 20000))
    scale = np.where(w < 2.0 ** -12, 2.0 ** 20, 64.0)
    rest = (w * scale).astype(np.float16).astype(np.float64)
    total = np.zeros_like(w)
    for i in range(3):
        part = E4M3[to_e4m3(rest)]
        total += part / 16.0 ** i
        rest = (rest - part) * 16
    off = np.abs(total / scale - w)
    # fp16 (2^-11, or half of 2^-24), then the terms (2^-12, or half of 2^-9 / 256), of 2^20 w where
    # the smallest steps count
    assert (off <= w * (2.0 ** -12 + F16_STEP) + (2.0 ** -25 + 2.0 ** -18) / 2.0 ** 20).all()
