"""Packed attention, rotated cache append and paged attention against plain float64 forms.

Tolerances, from the formats: with u = finfo(dtype).eps / 2 a result o = sum_j w_j v_j / l differs by
  u |o|                 its own rounding,
  u A                   the rounding of the weights w_j (A = sum_j w_j |v_j| / l),
  2 d A                 the scores' error d = D 2^-22 scale max_j sum_c |q_c k_jc| (f32 products; the
                        tensor cores truncate, hence two bits), in w_j and in l,
  2^-16 A               exp2, the products' and l's f32 sums over at most 2^13 keys here,
  n 2^-25 max|v| / l    float16 weights below 2^-14 (steps of 2^-24), relative to the largest, 1,
  2^-25                 a float16 result below 2^-14.
The log-sum differs by d + n 2^-24 + 2^-20 + 2^-23 |lse|. A rotation differs by u |y| + 2^-22 (|a| +
|b|) (+ 2^-25 in float16).
"""
import math
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import dinov3_b200 as dv  # noqa: E402

DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
both = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
dims = pytest.mark.parametrize("dim", [64, 128])


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def cu_of(lengths):
    return ints([0] + list(torch.tensor(lengths).cumsum(0))) if lengths else ints([0])


def one_sequence(q, k, v, scale, causal):
    """(out, its tolerance, lse, its tolerance) of one sequence in float64."""
    a, hq, d = q.shape
    b, hkv, _ = k.shape
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    qd, kd, vd = q.double(), k.double().repeat_interleave(hq // hkv, 1), v.double().repeat_interleave(hq // hkv, 1)
    seen = torch.arange(b, device=DEV)[None, :] <= torch.arange(a, device=DEV)[:, None] + (b - a if causal else b)
    s = torch.einsum("ihd,jhd->hij", qd, kd) * scale
    big = torch.einsum("ihd,jhd->hij", qd.abs(), kd.abs()) * scale
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if b else s.new_full((hq, a, 1), -math.inf)
    w = torch.exp(s - top.clamp(min=-1e300)).masked_fill(~seen, 0.0)
    total = w.sum(-1, keepdim=True)
    some = total.clamp(min=1e-300)
    o = torch.einsum("hij,jhd->ihd", w / some, vd)
    mean_abs = torch.einsum("hij,jhd->ihd", w / some, vd.abs())
    err = d * 2.0 ** -22 * (big.masked_fill(~seen, 0.0).amax(-1) if b else big.new_zeros(hq, a))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    lead = (b * tiny * (vd.abs().amax() if b else 0.0) / some[..., 0]).T[..., None]
    tol = u * o.abs() + (u + 2 * err.T[..., None] + 2.0 ** -16) * mean_abs + lead * (total[..., 0].T[..., None] > 0) + tiny
    lse = (top[..., 0] + total[..., 0].log()).T
    lse_tol = err.T + b * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -23 * lse.abs().nan_to_num(posinf=0.0)
    return o, tol, lse, lse_tol


def check(got, want, tol, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    bad &= ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp(min=1e-30))[bad].max()):.2f} of the tolerance"


def check_packed(q, k, v, out, lse, len_q, len_k, causal, scale, first_q=0, first_k=0):
    tq, tk = first_q, first_k
    for i, (a, b) in enumerate(zip(len_q, len_k)):
        o, tol, l, ltol = one_sequence(q[tq:tq + a], k[tk:tk + b], v[tk:tk + b], scale, causal)
        check(out[tq:tq + a], o, tol, f"sequence {i}")
        if lse is not None:
            check(lse[tq:tq + a], l, ltol, f"log-sum of sequence {i}")
        tq, tk = tq + a, tk + b


def packed_case(seed, len_q, len_k, hq, hkv, dim, dtype, spread=1.0):
    g = gen(seed)
    q = randn(g, sum(len_q), hq, dim, dtype=dtype) * spread
    k, v = (randn(g, sum(len_k), hkv, dim, dtype=dtype) for _ in range(2))
    return q, k, v


# ---- packed attention ------------------------------------------------------------------------
LENGTHS = [
    ([1], [1]),
    ([2, 1, 3], None),
    ([127, 128, 129], None),
    ([201, 201], None),
    ([0, 5, 0, 300, 0], None),
    ([255, 256, 257, 64], None),
    ([700], None),
    ([1, 1, 1], [1, 129, 1000]),            # one new token behind cached ones
    ([33, 100, 7], [400, 100, 135]),        # chunks behind cached keys
    ([50, 10], [20, 0]),                    # more queries than keys: rows without any key
    ([130, 300], [1, 129]),
]


@pytest.mark.parametrize("len_q,len_k", LENGTHS)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@dims
@both
def test_packed_lengths(len_q, len_k, causal, dim, dtype):
    len_k = len_k or len_q
    q, k, v = packed_case(1, len_q, len_k, 4, 2, dim, dtype, 2.0)
    lse = torch.full((q.shape[0], 4), 7.0, device=DEV)
    out = dv.attention_packed(q, k, v, cu_of(len_q), cu_of(len_k), causal=causal, lse=lse)
    check_packed(q, k, v, out, lse, len_q, len_k, causal, dim ** -0.5)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 6), (3, 1), (5, 1), (14, 2), (16, 1), (24, 2), (40, 1), (128, 1)])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@both
def test_packed_head_groups(hq, hkv, causal, dtype):
    len_q = [70, 3, 150]
    q, k, v = packed_case(2, len_q, len_q, hq, hkv, 64, dtype)
    lse = torch.empty(q.shape[0], hq, device=DEV)
    out = dv.attention_packed(q, k, v, cu_of(len_q), causal=causal, lse=lse, scale=0.3)
    check_packed(q, k, v, out, lse, len_q, len_q, causal, 0.3)


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@dims
def test_packed_long(causal, dim):
    len_q, len_k = [2048, 1500], [2048, 3001]
    q, k, v = packed_case(3, len_q, len_k, 4, 1, dim, torch.bfloat16, 3.0)
    out = dv.attention_packed(q, k, v, cu_of(len_q), cu_of(len_k), causal=causal)
    check_packed(q, k, v, out, None, len_q, len_k, causal, dim ** -0.5)


@pytest.mark.parametrize("len_q,len_k", [([1], [5000]), ([70, 3], [3000, 1500]), ([300, 0, 10, 64], [2500, 700, 5, 2048]), ([1030], [1030]), ([600, 1], [20, 4000])])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (6, 6), (5, 1)])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@both
def test_packed_few_queries_many_keys(len_q, len_k, hq, hkv, causal, dtype):
    """Long items are cut into parts for several CTAs and joined."""
    for dim in (64, 128):
        q, k, v = packed_case(12, len_q, len_k, hq, hkv, dim, dtype, 2.0)
        lse = torch.empty(q.shape[0], hq, device=DEV)
        status = torch.zeros(2, dtype=torch.int32, device=DEV)
        scratch = torch.full((1 << 26,), 255, dtype=torch.uint8, device=DEV)  # NaN wherever it is not written
        out = dv.attention_packed(q, k, v, cu_of(len_q), cu_of(len_k), causal=causal, lse=lse, workspace=scratch, status=status)
        check_packed(q, k, v, out, lse, len_q, len_k, causal, dim ** -0.5)
        assert torch.equal(out, dv.attention_packed(q, k, v, cu_of(len_q), cu_of(len_k), causal=causal)) and status.tolist() == [0, 0]


def test_packed_cut_items_and_values_that_are_not_finite():
    """A part at the diagonal keeps later keys' infinities from the rows that do not see them."""
    q, k, v = packed_case(13, [100], [3000], 4, 2, 64, torch.float16)
    want = dv.attention_packed(q, k, v, ints([0, 100]), ints([0, 3000]), causal=True)
    v2 = v.clone()
    v2[2950:] = math.inf
    got = dv.attention_packed(q, k, v2, ints([0, 100]), ints([0, 3000]), causal=True)
    assert torch.equal(got[:50], want[:50]) and (got[50:] == math.inf).all()


@both
def test_packed_many_sequences(dtype):
    rng = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 60, (1500,), generator=rng).tolist()
    q, k, v = packed_case(4, lens, lens, 2, 1, 64, dtype)
    out = dv.attention_packed(q, k, v, cu_of(lens), causal=True)
    check_packed(q, k, v, out, None, lens, lens, True, 0.125)


@both
@dims
def test_packed_strides(dtype, dim):
    """Fused rows, head-major tensors, and an output inside a wider one."""
    lens, g = [201, 30, 77], gen(6)
    t, cu = sum(lens), cu_of(lens)
    qkv = randn(g, t, 12, dim, dtype=dtype)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    wide = torch.full((t, 9, dim + 16), 3.0, device=DEV, dtype=dtype)
    out = dv.attention_packed(q, k, v, cu, causal=True, out=wide[:, 1:, 8:8 + dim])
    check_packed(q, k, v, out, None, lens, lens, True, dim ** -0.5)
    assert (wide[:, 0] == 3.0).all() and (wide[:, :, :8] == 3.0).all() and (wide[:, :, 8 + dim:] == 3.0).all()
    q2, k2, v2 = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    out2 = dv.attention_packed(q2, k2, v2, cu, causal=True, out=torch.empty(8, t, dim, device=DEV, dtype=dtype).transpose(0, 1))
    assert torch.equal(out, out2)


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@both
def test_packed_rows_outside_are_left(dtype, causal):
    q, k, v = packed_case(7, [300], [300], 2, 2, 64, dtype)
    out = torch.full_like(q, 5.0)
    lse = torch.full((300, 2), 5.0, device=DEV)
    cu = ints([10, 60, 60, 270])
    dv.attention_packed(q, k, v, cu, causal=causal, out=out, lse=lse)
    check_packed(q, k, v, out, lse, [50, 0, 210], [50, 0, 210], causal, 0.125, 10, 10)
    for x in (out, lse):
        assert (x[:10] == 5.0).all() and (x[270:] == 5.0).all()
    # bounds outside the tensors are clamped to them
    out = dv.attention_packed(q, k, v, ints([-5, 100, 99999]), causal=causal, out=torch.full_like(q, 5.0))
    check_packed(q, k, v, out, None, [100, 200], [100, 200], causal, 0.125)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@dims
@both
def test_packed_unseen_rows_do_not_reach_a_result(dtype, dim, bad):
    """NaN and infinities in the rows behind a sequence, in its neighbours and, causal, in later
    keys."""
    lens = [100, 37, 190]
    q, k, v = packed_case(8, [sum(lens) + 20], [sum(lens) + 20], 4, 2, dim, dtype)
    cu = cu_of(lens)
    want = dv.attention_packed(q, k, v, cu)
    k2, v2 = k.clone(), v.clone()
    k2[100:137], v2[100:137], k2[327:], v2[327:] = bad, bad, bad, bad
    got = dv.attention_packed(q, k2, v2, cu)
    assert torch.equal(got[:100], want[:100]) and torch.equal(got[137:327], want[137:327])
    want = dv.attention_packed(q, k, v, cu, causal=True)
    k2, v2 = k.clone(), v.clone()
    k2[60:100], v2[60:100, 0], v2[300:327] = bad, bad, bad
    got = dv.attention_packed(q, k2, v2, cu, causal=True)
    assert torch.equal(got[:60], want[:60]) and torch.equal(got[100:300], want[100:300])
    # the keys that are seen do reach it: infinite values of v where only v is infinite
    o, tol, _, _ = one_sequence(q[137:327], k[137:327], v2[137:327].nan_to_num(0.0, 0.0, 0.0), dim ** -0.5, True)
    hit = got[300:327].double()
    assert (hit.isnan() if math.isnan(bad) else hit == bad).all()


@dims
def test_packed_bad_queries_stay_in_their_rows(dim):
    q, k, v = packed_case(14, [150, 60], [150, 60], 6, 2, dim, torch.bfloat16)
    cu = cu_of([150, 60])
    want = dv.attention_packed(q, k, v, cu, causal=True)
    q2 = q.clone()
    q2[77, 4], q2[160, 0] = math.nan, math.inf
    got = dv.attention_packed(q2, k, v, cu, causal=True)
    assert got[77, 4].isnan().all() and got[160, 0].isnan().all()
    got[77, 4], got[160, 0] = want[77, 4], want[160, 0]
    assert torch.equal(got, want)


@both
def test_packed_extreme_scores(dtype):
    """Scores far apart and of one sign, and equal ones: the maximum moves with almost every key."""
    n, g = 300, gen(9)
    q = torch.ones(n, 1, 64, device=DEV, dtype=dtype)
    v = randn(g, n, 1, 64, dtype=dtype)
    ramp = torch.arange(n, device=DEV, dtype=torch.float32)[:, None, None]
    for k in (ramp * 0.5 - 75, 75 - ramp * 0.5, torch.full_like(ramp, -900.0), torch.full_like(ramp, 900.0), torch.zeros_like(ramp)):
        k = (k.expand(n, 1, 64) * torch.ones(64, device=DEV)).to(dtype).contiguous()
        lse = torch.empty(n, 1, device=DEV)
        out = dv.attention_packed(q, k, v, ints([0, n]), causal=True, lse=lse)
        check_packed(q, k, v, out, lse, [n], [n], True, 0.125)


def test_packed_capture_and_replay():
    """A captured call follows its inputs and its bounds; two streams at once; the same bits."""
    q, k, v = packed_case(10, [600], [600], 4, 2, 128, torch.bfloat16)
    cu = ints([0, 200, 600])
    eager = dv.attention_packed(q, k, v, cu, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = dv.attention_packed(q, k, v, cu, causal=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = dv.attention_packed(q, k, v, cu, causal=True)
    side.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager) and torch.equal(held, eager)
    cu.copy_(ints([0, 451, 600]))
    q.copy_(q.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    check_packed(q, k, v, held, None, [451, 149], [451, 149], True, 128 ** -0.5)


def test_packed_nothing_to_do():
    q = torch.empty(0, 4, 64, device=DEV, dtype=torch.float16)
    assert dv.attention_packed(q, q, q, ints([0])).shape == q.shape
    assert dv.attention_packed(q, q, q, ints([0, 0, 0]), causal=True).shape == q.shape
    q1 = torch.ones(3, 4, 64, device=DEV, dtype=torch.float16)
    assert (dv.attention_packed(q1, q, q, ints([0, 3]), ints([0, 0])) == 0).all()


# ---- the cache -------------------------------------------------------------------------------
@dims
def test_packed_empty_tensors_with_strides_of_nothing(dim):
    """[heads, 0, dim] seen as [0, heads, dim] has a head stride of 0."""
    none = torch.empty(4, 0, dim, device=DEV, dtype=torch.float16).transpose(0, 1)
    q, cu, some = randn(gen(16), 5, 4, dim, dtype=torch.float16), ints([0, 0, 0]), ints([0, 2, 5])
    assert dv.attention_packed(none, q, q, cu, some).shape == (0, 4, dim)
    assert (dv.attention_packed(q, none, none, some, cu) == 0).all()
    assert dv.attention_packed(none, none, none, cu).shape == (0, 4, dim)


def paged_cache(seed, lens, hkv, page, dim, dtype, wide=0, joined=False):
    """A shuffled table (unused entries -1) over random pages; `joined`: k and v in one pool."""
    g = gen(seed)
    counts = [-(-max(n, 0) // page) for n in lens]
    pool = sum(counts) + 2
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(counts + [1]) + wide), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    if joined:
        kv = randn(g, pool, 2, hkv, page, dim, dtype=dtype)
        return kv[:, 0], kv[:, 1], table
    return randn(g, pool, hkv, page, dim, dtype=dtype), randn(g, pool, hkv, page, dim, dtype=dtype), table


def cached_rows(cache, table, i, n):
    page = cache.shape[2]
    ids = table[i, :-(-n // page)].long()
    return cache[ids].transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:n]


def check_paged(q, k, v, table, lens, out, lse, scale):
    for i, n in enumerate(lens):
        n = max(n, 0)
        o, tol, l, ltol = one_sequence(q[i:i + 1], cached_rows(k, table, i, n), cached_rows(v, table, i, n), scale, False)
        check(out[i:i + 1], o, tol, f"sequence {i}")
        if lse is not None:
            check(lse[i:i + 1], l, ltol, f"log-sum of sequence {i}")


@pytest.mark.parametrize("page", [1, 7, 16, 64, 100, 256])
@dims
@both
def test_paged_lengths(page, dim, dtype):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 500, 1025, -3]
    k, v, table = paged_cache(20, lens, 2, page, dim, dtype, wide=1)
    q = randn(gen(21), len(lens), 8, dim, dtype=dtype) * 2
    lse = torch.empty(len(lens), 8, device=DEV)
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    out = dv.attention_paged(q, k, v, table, ints(lens), lse=lse, status=status)
    check_paged(q, k, v, table, lens, out, lse, dim ** -0.5)
    assert status.tolist() == [0, 0]


@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 6), (3, 1), (14, 2), (16, 2), (16, 1), (20, 1), (33, 1), (128, 1), (7, 7)])
@dims
def test_paged_head_groups(hq, hkv, dim):
    lens = [300, 1, 77]
    for dtype in TYPES.values():
        k, v, table = paged_cache(22, lens, hkv, 16, dim, dtype)
        q = randn(gen(23), 3, hq, dim, dtype=dtype)
        lse = torch.empty(3, hq, device=DEV)
        out = dv.attention_paged(q, k, v, table, ints(lens), lse=lse, scale=0.2)
        check_paged(q, k, v, table, lens, out, lse, 0.2)


@pytest.mark.parametrize("max_len", [1, 64, 5000, None])
@both
def test_paged_long_and_any_bound(max_len, dtype):
    """The bound of the lengths decides the split, not the result."""
    lens = [5000, 8000, 3, 0, 4096]
    k, v, table = paged_cache(24, lens, 1, 32, 128, dtype, joined=True)
    q = randn(gen(25), len(lens), 4, 128, dtype=dtype) * 3
    lse = torch.empty(len(lens), 4, device=DEV)
    out = dv.attention_paged(q, k, v, table, ints(lens), max_len=max_len, lse=lse)
    check_paged(q, k, v, table, lens, out, lse, 128 ** -0.5)
    again = dv.attention_paged(q, k, v, table, ints(lens), max_len=max_len)
    assert torch.equal(out, again)


@pytest.mark.parametrize("hq,hkv", [(4, 2), (33, 1), (8, 8)])
@pytest.mark.parametrize("lens", [[300], [257, 0], [1100, 300, 5], [700] * 9, [400, 1] * 12])
@both
@dims
def test_paged_few_sequences(lens, hq, hkv, dtype, dim):
    """Few units of medium length, whose blocks meet in a cluster; bounds below the lengths too."""
    k, v, table = paged_cache(28, lens, hkv, 16, dim, dtype)
    q, lse = randn(gen(29), len(lens), hq, dim, dtype=dtype) * 2, torch.empty(len(lens), hq, device=DEV)
    for max_len in (None, 270):
        out = dv.attention_paged(q, k, v, table, ints(lens), max_len=max_len, lse=lse.fill_(7.0))
        check_paged(q, k, v, table, lens, out, lse, dim ** -0.5)


@pytest.mark.parametrize("hq,hkv,longest", [(4, 2, 700), (33, 1, 400), (3, 3, 2000)])
@dims
def test_paged_many_sequences(hq, hkv, longest, dim):
    """More sequences than a block has threads, empty ones among them, in a workspace that holds NaN."""
    g = gen(26 + dim)
    lens = torch.randint(0, longest, (300,), generator=g, device=DEV).tolist()
    lens[:3], lens[100:104], lens[-2:] = [0, 0, longest], [0, 0, 0, 1], [longest, 0]
    k, v, table = paged_cache(27, lens, hkv, 16, dim, torch.bfloat16)
    q, lse = randn(g, len(lens), hq, dim, dtype=torch.bfloat16), torch.empty(len(lens), hq, device=DEV)
    out = dv.attention_paged(q, k, v, table, ints(lens), lse=lse, workspace=torch.full((1 << 26,), 255, dtype=torch.uint8, device=DEV))
    check_paged(q, k, v, table, lens, out, lse, dim ** -0.5)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@dims
@both
def test_paged_unused_slots_do_not_reach_a_result(dtype, dim, bad):
    lens = [1, 17, 40, 129]
    k, v, table = paged_cache(26, lens, 2, 16, dim, dtype)
    q = randn(gen(27), 4, 8, dim, dtype=dtype)
    want = dv.attention_paged(q, k, v, table, ints(lens))
    k2, v2 = torch.full_like(k, bad), torch.full_like(v, bad)
    for i, n in enumerate(lens):
        for j in range(n):
            k2[table[i, j // 16], :, j % 16] = k[table[i, j // 16], :, j % 16]
            v2[table[i, j // 16], :, j % 16] = v[table[i, j // 16], :, j % 16]
    assert torch.equal(dv.attention_paged(q, k2, v2, table, ints(lens)), want)


@both
def test_paged_bad_pages_are_reported(dtype):
    """A page outside the pool counts as absent and sets the bit; so does a length past the table."""
    lens = [100, 100, 100, 100]
    k, v, table = paged_cache(28, lens, 1, 16, 64, dtype)
    q = randn(gen(29), 4, 2, 64, dtype=dtype)
    want = dv.attention_paged(q, k, v, table, ints(lens))
    broken = table.clone()
    broken[1, 2], broken[2, 0] = -1, k.shape[0]
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    out = dv.attention_paged(q, k, v, broken, ints(lens), status=status)
    assert status.tolist() == [1 << 6, 0]
    assert torch.equal(out[0], want[0]) and torch.equal(out[3], want[3])
    keep = torch.cat([torch.arange(32), torch.arange(48, 100)]).to(DEV)
    for i, rows in ((1, keep), (2, torch.arange(16, 100, device=DEV))):
        o, tol, _, _ = one_sequence(q[i:i + 1], cached_rows(k, table, i, 100)[rows], cached_rows(v, table, i, 100)[rows], 0.125, False)
        check(out[i:i + 1], o, tol)
    status.zero_()
    out = dv.attention_paged(q, k, v, table, ints([100, 100, 113, 2**31 - 1]), status=status)
    assert status.tolist()[0] == 1 << 6 and torch.equal(out[:2], want[:2])
    status.zero_()
    all_bad = torch.full_like(table, 2**30)
    assert (dv.attention_paged(q, k, v, all_bad, ints(lens), status=status) == 0).all() and status.tolist()[0] == 1 << 6


def test_paged_offsets_past_32_bits():
    """Pages whose element offset passes 2^32."""
    page, hkv, dim = 64, 8, 128
    pages = (1 << 32) // (page * hkv * dim) + 4
    k = torch.empty(pages, hkv, page, dim, device=DEV, dtype=torch.float16)
    v = torch.empty_like(k)
    g = gen(30)
    ids = [pages - 1, 5, pages - 3]
    for i in ids:
        k[i], v[i] = randn(g, hkv, page, dim, dtype=torch.float16), randn(g, hkv, page, dim, dtype=torch.float16)
    table, lens = ints([ids, ids]), [190, 65]
    q = randn(g, 2, 32, dim, dtype=torch.float16)
    new_k, new_v = randn(g, 2, hkv, dim, dtype=torch.float16), randn(g, 2, hkv, dim, dtype=torch.float16)
    dv.rope_append(None, new_k[:1], new_v[:1], k, v, table[:1], ints([191]))
    assert torch.equal(k[pages - 3, :, 62], new_k[0]) and torch.equal(v[pages - 3, :, 62], new_v[0])
    out = dv.attention_paged(q, k, v, table, ints([191, 65]))
    check_paged(q, k, v, table, [191, 65], out, None, dim ** -0.5)


def test_paged_capture_streams_and_workspace():
    lens = [3000, 17, 900]
    k, v, table = paged_cache(31, lens, 2, 16, 128, torch.bfloat16)
    q = randn(gen(32), 3, 8, 128, dtype=torch.bfloat16)
    n = ints(lens)
    eager = dv.attention_paged(q, k, v, table, n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [dv.attention_paged(q, k, v, table, n) for _ in range(8)]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    for g in graphs:
        with torch.cuda.graph(g):
            held.append(dv.attention_paged(q, k, v, table, n))
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, eager) for o in outs + held)
    n.copy_(ints([2999, 1, 64]))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for h in held:
        check_paged(q, k, v, table, [2999, 1, 64], h, None, 128 ** -0.5)
    given = dv.attention_paged(q, k, v, table, n, workspace=torch.full((1 << 24,), 255, dtype=torch.uint8, device=DEV))
    assert torch.equal(given, held[0])
    assert dv.attention_paged(q[:0], k, v, table[:0], n[:0]).shape == (0, 8, 128)


FIRST_CALL = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, dinov3_b200 as dv
d = "cuda:0"
q = torch.randn(40, 8, 64, device=d).half()
cache, table = torch.zeros(80, 8, 16, 64, device=d).half(), torch.arange(80, dtype=torch.int32, device=d).view(1, 80)
cu, n = torch.tensor([0, 40], dtype=torch.int32, device=d), torch.tensor([1200], dtype=torch.int32, device=d)
cos = torch.ones(1300, 32, device=d)
big = torch.randn(4096, 8, 64, device=d).half()
big_cu = torch.tensor([0, 4096], dtype=torch.int32, device=d)
def step():
    a = dv.attention_packed(q, q, q, cu)
    b = dv.attention_packed(q, big, big, cu, big_cu, causal=True)
    r = dv.rope_append(q, q, q, cache, cache.clone(), table, n, cos, cos, cu_new=cu)
    return a, b, r, dv.attention_paged(q[:1], cache, cache, table, n)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    held = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(held, step()))
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture():
    here = os.path.dirname(os.path.abspath(__file__))
    got = subprocess.run([sys.executable, "-c", FIRST_CALL, os.path.join(os.path.dirname(here), "dinov3-loom_b200")], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "same", got.stderr[-2000:]


# ---- append ----------------------------------------------------------------------------------
def tables(positions, rot):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return angle.cos().float().to(DEV), angle.sin().float().to(DEV)


def rotated(x, cos, sin):
    """(y, tolerance) of the rows x at the tables' rows, in float64."""
    half = cos.shape[-1]
    xd, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b, rest = xd[..., :half], xd[..., half:2 * half], xd[..., 2 * half:]
    y = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    size = a.abs() + b.abs()
    tol = y.abs() * (torch.finfo(x.dtype).eps / 2) + 2.0 ** -22 * torch.cat([size, size, torch.zeros_like(rest)], -1)
    return y, tol + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("new,held", [([1], [0]), ([3, 1, 40], [0, 100, 15]), ([0, 33, 0, 1], [5, 31, 0, 64]), ([1, 1, 1, 1], [0, 15, 16, 77]), ([300, 2], [0, 1])])
@pytest.mark.parametrize("page", [1, 16, 48])
@pytest.mark.parametrize("hq,hkv,dim,rot", [(8, 2, 64, 64), (6, 6, 64, 32), (5, 1, 128, 128), (12, 4, 128, 48), (4, 4, 64, 0)])
@both
def test_append(new, held, page, hq, hkv, dim, rot, dtype):
    total = [a + b for a, b in zip(new, held)]
    k_cache, v_cache, table = paged_cache(40, total, hkv, page, dim, dtype, joined=True)
    k0, v0 = k_cache.clone(), v_cache.clone()
    g, t = gen(41), sum(new)
    qkv = randn(g, t + 3, hq + 2 * hkv, dim, dtype=dtype)  # three rows behind the last sequence
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cos, sin = tables(400, rot) if rot else (None, None)
    q_out = torch.full((t + 3, hq, dim), 9.0, device=DEV, dtype=dtype)
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    dv.rope_append(q, k, v, k_cache, v_cache, table, ints(total), cos, sin, cu_new=cu_of(new), q_out=q_out, status=status)
    assert status.tolist() == [0, 0] and (q_out[t:] == 9.0).all()
    at = 0
    for i, (a, b) in enumerate(zip(new, total)):
        pos = torch.arange(b - a, b, device=DEV)
        ids, slot = table[i].long()[pos // page], pos % page
        for got, x in ((q_out[at:at + a], q[at:at + a]), (k_cache[ids, :, slot], k[at:at + a])):
            if rot:
                check(got, *rotated(x, cos[pos], sin[pos]))
            else:
                assert torch.equal(got, x)
        assert torch.equal(v_cache[ids, :, slot], v[at:at + a])
        k0[ids, :, slot], v0[ids, :, slot] = k_cache[ids, :, slot], v_cache[ids, :, slot]
        at += a
    assert torch.equal(k0, k_cache) and torch.equal(v0, v_cache)  # nothing else was written
    if all(a == 1 for a in new):  # the form for one row each, and in place
        k1, v1, mine = k_cache.clone(), v_cache.clone(), q[:t].clone()
        back = dv.rope_append(mine, k[:t], v[:t], k1, v1, table, ints(total), cos, sin, q_out=mine)
        assert back is mine and torch.equal(mine, q_out[:t]) and torch.equal(k1, k_cache) and torch.equal(v1, v_cache)


@both
def test_append_many_sequences(dtype):
    rng = torch.Generator().manual_seed(11)
    new = torch.randint(0, 4, (1300,), generator=rng).tolist()
    k_cache, v_cache, table = paged_cache(42, new, 1, 4, 64, dtype)
    k, v = randn(gen(43), sum(new), 1, 64, dtype=dtype), randn(gen(44), sum(new), 1, 64, dtype=dtype)
    assert dv.rope_append(None, k, v, k_cache, v_cache, table, ints(new), cu_new=cu_of(new)) is None
    at = 0
    for i, n in enumerate(new):
        if n:
            assert torch.equal(k_cache[table[i, 0], :, :n].transpose(0, 1), k[at:at + n])
            assert torch.equal(v_cache[table[i, 0], :, :n].transpose(0, 1), v[at:at + n])
        at += n


def test_append_skips_and_reports_bad_places():
    new, total = [4, 4, 4, 4], [4, 20, 4, 3]
    k_cache, v_cache, table = paged_cache(45, [20] * 4, 2, 8, 64, torch.float16)
    table[0, 0], table[1, 2] = k_cache.shape[0], -1
    k0 = k_cache.clone()
    q, k, v = (randn(gen(46), 16, 2, 64, dtype=torch.float16) for _ in range(3))
    cos, sin = tables(18, 64)
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    q_out = torch.full_like(q, 9.0)
    dv.rope_append(q, k, v, k_cache, v_cache, table, ints(total), cos, sin, cu_new=cu_of(new), q_out=q_out, status=status)
    assert status.tolist() == [3 << 6, 0]
    # sequence 1: positions 16, 17 lie on a bad page, 18 and 19 behind the tables; sequence 3 starts at -1
    assert (q_out[6:8] == 9.0).all() and (q_out[12] == 9.0).all() and not (q_out[4:6] == 9.0).any()
    good = table[2, 0]
    assert not torch.equal(k_cache[good, :, :4], k0[good, :, :4])
    k_cache[good, :, :4] = k0[good, :, :4]
    k_cache[table[3, 0], :, :3] = k0[table[3, 0], :, :3]
    assert torch.equal(k_cache, k0)
    # positions behind the page table
    status.zero_()
    dv.rope_append(None, k[:4], v[:4], k_cache, v_cache, table, ints([1, 10**6, 2**31 - 1, 25]), status=status)
    assert status.tolist() == [1 << 6, 0]


# ---- together --------------------------------------------------------------------------------
@both
@dims
def test_calls_that_read_what_the_one_before_wrote(dtype, dim):
    """A launch may be set up under the end of the one before. Layers whose every call reads the output
    of the call before it, with one workspace for all: the same bits whether the host waits between
    the calls, does not, or replays them from a graph."""
    hq, hkv, page, lens = 8, 2, 16, [1, 900, 37, 2100, 0, 300]
    g, rows = gen(60 + dim), sum(lens)
    k_cache, v_cache, table = paged_cache(61, lens, hkv, page, dim, dtype)
    first = randn(g, rows, hq, dim, dtype=dtype)
    cos, sin = tables(4096, dim)
    cu, n = cu_of(lens), ints(lens)
    scratch = torch.empty(1 << 27, dtype=torch.uint8, device=DEV)

    def layers(wait):
        x, got = first, []
        for _ in range(5):
            q = dv.rope_append(x, x[:, :hkv], x[:, hkv:2 * hkv], k_cache, v_cache, table, n, cos, sin, cu_new=cu)
            wait()
            x = dv.attention_packed(q, q[:, :hkv], q[:, hkv:2 * hkv], cu, causal=True, workspace=scratch)
            wait()
            got += [q, x, dv.attention_paged(x[:len(lens)], k_cache, v_cache, table, n, workspace=scratch)]
            wait()
        return got

    waited = [t.clone() for t in layers(torch.cuda.synchronize)]
    assert waited[-1].abs().max() > 0 and not torch.equal(waited[1], waited[4])
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(waited, layers(lambda: None)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layers(lambda: None)
    for _ in range(2):
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(waited, held))


@both
def test_prompt_then_tokens(dtype):
    """A decoder's attention: prompts packed, rotated, cached and attended, then tokens one at a
    time, against the whole sequences in float64. Captured decode steps give the eager bits."""
    hq, hkv, dim, page, steps = 8, 2, 64, 16, 5
    lens, g = [37, 1, 130], gen(50)
    whole = [n + steps for n in lens]
    k_cache, v_cache, table = paged_cache(51, whole, hkv, page, dim, dtype)
    rows = [randn(g, n, hq + 2 * hkv, dim, dtype=dtype) for n in whole]
    cos, sin = tables(256, dim)
    cu, n = cu_of(lens), ints(lens)
    prompt = torch.cat([r[:m] for r, m in zip(rows, lens)])
    q = dv.rope_append(prompt[:, :hq], prompt[:, hq:hq + hkv], prompt[:, hq + hkv:], k_cache, v_cache, table, n, cos, sin, cu_new=cu)
    keys = torch.cat([cached_rows(k_cache, table, i, m) for i, m in enumerate(lens)])
    out = dv.attention_packed(q, keys, prompt[:, hq + hkv:], cu, causal=True)
    outs, qs = [[o] for o in out.split(lens)], [[x] for x in q.split(lens)]
    new = torch.empty(3, hq + 2 * hkv, dim, device=DEV, dtype=dtype)

    def step():
        q = dv.rope_append(new[:, :hq], new[:, hq:hq + hkv], new[:, hq + hkv:], k_cache, v_cache, table, n, cos, sin)
        return q, dv.attention_paged(q, k_cache, v_cache, table, n, max_len=192)

    graph = torch.cuda.CUDAGraph()
    new.zero_()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(steps):
        new.copy_(torch.stack([r[m + i] for r, m in zip(rows, lens)]))
        n.add_(1)
        got = step()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, got))
        for j in range(3):
            qs[j].append(got[0][j:j + 1])
            outs[j].append(got[1][j:j + 1])
    for i, m in enumerate(whole):
        q, keys = torch.cat(qs[i]), cached_rows(k_cache, table, i, m)
        check(q, *rotated(rows[i][:, :hq], cos[:m], sin[:m]))
        check(keys, *rotated(rows[i][:, hq:hq + hkv], cos[:m], sin[:m]))
        o, tol, _, _ = one_sequence(q, keys, rows[i][:, hq + hkv:], dim ** -0.5, True)
        check(torch.cat(outs[i]), o, tol)


def test_refusals_of_tensors():
    """What the Python face refuses before it launches anything."""
    q = torch.zeros(4, 4, 64, device=DEV, dtype=torch.float16)
    cu, n = ints([0, 4]), ints([4])
    cache, table = torch.zeros(2, 4, 8, 64, device=DEV, dtype=torch.float16), ints([[0, 1]])
    calls = [
        lambda: dv.attention_packed(q.float(), q.float(), q.float(), cu),
        lambda: dv.attention_packed(q.cpu(), q.cpu(), q.cpu(), cu),
        lambda: dv.attention_packed(q, q.bfloat16(), q, cu),
        lambda: dv.attention_packed(q, q[:, :3], q[:, :3], cu),
        lambda: dv.attention_packed(q, q, q[:3], cu),
        lambda: dv.attention_packed(q[..., :32], q[..., :32], q[..., :32], cu),
        lambda: dv.attention_packed(q, q, q, cu.long()),
        lambda: dv.attention_packed(q, q, q, cu, ints([0, 1, 4])),
        lambda: dv.attention_packed(q, q, q, cu, scale=0.0),
        lambda: dv.attention_packed(q, q, q, cu, scale=math.nan),
        lambda: dv.attention_packed(q, q, q, cu, out=q[:3].clone()),
        lambda: dv.attention_packed(q, q, q, cu, out=torch.zeros(4, 1, 64, device=DEV, dtype=torch.float16).expand(4, 4, 64)),
        lambda: dv.attention_packed(q, q[:, :1].expand(4, 4, 64), q, cu),
        lambda: dv.attention_packed(q, q, q, cu, lse=torch.zeros(4, 3, device=DEV)),
        lambda: dv.attention_packed(torch.zeros(4, 4, 65, device=DEV, dtype=torch.float16)[..., 1:], q, q, cu),
        lambda: dv.attention_packed(q.clone().requires_grad_(), q, q, cu),
        lambda: dv.rope_append(q, q, q, cache, cache.clone(), table, n),
        lambda: dv.rope_append(q, q, q, cache, cache[:, :2], table, n, cu_new=cu),
        lambda: dv.rope_append(q, q, q, cache.transpose(1, 2), cache, table, n, cu_new=cu),
        lambda: dv.rope_append(q, q, q, cache, cache, table, n, torch.zeros(9, 20, device=DEV), torch.zeros(9, 20, device=DEV), cu_new=cu),
        lambda: dv.rope_append(q, q, q, cache, cache, table, n, torch.zeros(9, 32, device=DEV), cu_new=cu),
        lambda: dv.rope_append(q, q, q, cache, cache, table, ints([4, 4]), cu_new=cu),
        lambda: dv.attention_paged(q[:1], cache, cache, table.long(), n),
        lambda: dv.attention_paged(q[:2], cache, cache, table, n),
        lambda: dv.attention_paged(q[:1], cache, cache, table, n, max_len=-1),
        lambda: dv.attention_paged(q[:1, :3], cache, cache, table, n),
        lambda: dv.attention_paged(q[:1], cache.bfloat16(), cache, table, n),
        lambda: dv.attention_paged(q[:1], cache, cache, table, n, status=torch.zeros(1, dtype=torch.int32, device=DEV)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(dv.DINOv3Error) as e:
            call()
        assert e.value.code == dv.INVALID_ARGUMENT, i
