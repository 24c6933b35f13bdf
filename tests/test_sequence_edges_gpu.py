"""Packed attention, rotated cache append and paged attention where their numbers and their arguments
reach an edge: scores beyond f32's integers, weights far below the largest, overlapping memory,
gradients that would be lost. Bounds are derived beside each test, with u = finfo(dtype).eps / 2.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import dinov3_b200 as dv  # noqa: E402
from test_sequence_gpu import DEV, both, cached_rows, check, cu_of, dims, gen, ints, one_sequence, paged_cache, randn  # noqa: E402


def fill_cache(keys, values, page, pool_seed):
    """Paged caches [pages, heads, page, dim] that hold the rows [n, heads, dim], and their table."""
    n, heads, dim = keys.shape
    k, v, table = paged_cache(pool_seed, [n], heads, page, dim, keys.dtype)
    pos = torch.arange(n, device=DEV)
    ids, slot = table[0].long()[pos // page], pos % page
    k[ids, :, slot], v[ids, :, slot] = keys, values
    return k, v, table


def every_form(q, k, v, scale):
    """(name, out, lse) of one query row over keys [n, heads, dim] by each way there is to ask for it."""
    n, hq = k.shape[0], q.shape[1]
    for name, causal in (("packed", False), ("packed causal", True)):
        lse = torch.empty(1, hq, device=DEV)
        out = dv.attention_packed(q, k, v, ints([0, 1]), ints([0, n]), causal=causal, scale=scale, lse=lse)
        yield name, out[0], lse[0]
    kc, vc, table = fill_cache(k, v, 16, 90)
    for max_len in (n, 256, 1 << 20):
        wide = torch.full((1, -(-max_len // 16)), -1, dtype=torch.int32, device=DEV)  # the table bounds max_len
        wide[:, :min(table.shape[1], wide.shape[1])] = table[:, :wide.shape[1]]
        if wide.shape[1] < table.shape[1]:
            wide = table
        lse = torch.empty(1, hq, device=DEV)
        out = dv.attention_paged(q, kc, vc, wide, ints([n]), max_len=max_len, scale=scale, lse=lse)
        yield f"paged, bound {max_len}", out[0], lse[0]


# ---- scores past f32's integers --------------------------------------------------------------
@pytest.mark.parametrize("n", [40, 300, 5000])
@pytest.mark.parametrize("order", ["up", "down", "twice"])
@dims
@both
def test_scores_far_beyond_one(n, order, dim, dtype):
    """q . k of 2^28 to 2^30 and 2^90 to 2^92, exact in f32 (one channel, short mantissas): the one largest score has
    all the weight, two equal ones half each. Any score differs from the largest by more than 2^20, so
    that the others' weights are exactly 0, and the result is that value, or the mean of two, rounded once."""
    g = gen(80)
    big = 2.0 ** 15 if dtype == torch.float16 else 2.0 ** 46
    hq, hkv = 6, 2
    steps = torch.arange(n, device=DEV) % 64
    x = (1 + steps / 64.0) if order == "up" else (2 - steps / 64.0)  # 7 bits
    x = x.clamp(max=1.9375)
    x[n // 3] = 1.96875  # the largest: 1 + 31/32
    if order == "twice":
        x[n - 2] = 1.96875
    k = torch.zeros(n, hkv, dim, device=DEV, dtype=dtype)
    k[:, :, 3] = (x * big / 2)[:, None].to(dtype)
    assert torch.equal(k[:, 0, 3].float(), x * big / 2)
    q = torch.zeros(1, hq, dim, device=DEV, dtype=dtype)
    q[0, :, 3] = (torch.tensor([1, 1.125, 1.25, 1.375, 1.5, 1.75], device=DEV) * big / 2).to(dtype)
    v = randn(g, n, hkv, dim, dtype=dtype)
    top = v[n // 3].double()
    if order == "twice":
        top = (top + v[n - 2].double()) / 2
    top = top.repeat_interleave(hq // hkv, 0)
    for scale in (1.0, 0.125, 777.0):
        score = q[0, :, 3].double() * (1.96875 * big / 2) * torch.tensor(scale, dtype=torch.float32).double().to(DEV)
        want_lse = score + (math.log(2.0) if order == "twice" else 0.0)
        for name, out, lse in every_form(q, k, v, scale):
            check(out, top, top.abs() * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 0.0), name)
            # scale log2(e), its product with the score and that with ln 2 are rounded to f32
            check(lse, want_lse, want_lse.abs() * 2.0 ** -21, name + ", log-sum")


@pytest.mark.parametrize("n", [300, 1000, 5000])
@pytest.mark.parametrize("scale", [1.0, 0.125])
@dims
@both
def test_large_scores_that_creep_up(n, scale, dim, dtype):
    """Scores near 2^29.8 that grow by one unit in the last place (64) every 128 keys: steps of 64 or 8
    (in the exponent of e) between groups of keys, where the product with scale log2(e) moves by less than
    its own rounding. The scores are exact in f32; of their differences' products 2^-22 is lost."""
    q, k = torch.zeros(1, 4, dim, device=DEV, dtype=dtype), torch.zeros(n, 2, dim, device=DEV, dtype=dtype)
    q[0, :, 3], k[:, :, 3] = 1.75 * 2.0 ** 14, 1.96875 * 2.0 ** 14
    step = torch.arange(n, device=DEV) // 128
    q[0, :, 9], k[:, :, 9] = 8.0, (8.0 * step)[:, None].to(dtype)
    v = randn(gen(81), n, 2, dim, dtype=dtype)
    s = step.double() * 64 * scale
    w = torch.exp(s - s.max())
    w /= w.sum()
    want = torch.einsum("j,jhd->hd", w, v.double()).repeat_interleave(2, 0)
    size = torch.einsum("j,jhd->hd", w, v.double().abs()).repeat_interleave(2, 0)
    u = torch.finfo(dtype).eps / 2
    for name, out, lse in every_form(q, k, v, scale):
        check(out, want, u * want.abs() + (u + 2.0 ** -16) * size + (2.0 ** -25 if dtype == torch.float16 else 0.0), name)


# ---- float16 weights far below the largest ---------------------------------------------------
@pytest.mark.parametrize("n,gap", [(300, 15.5), (8192, 15.5), (8192, 17.0), (8192, 19.0)])
@pytest.mark.parametrize("strong", ["first", "middle", "last"])
@dims
def test_many_weak_keys_beside_a_strong_one(n, gap, strong, dim):
    """One key of value 0 and n - 1 keys of value 1 whose scores lie `gap` below it, in float16: each weak
    weight is below the smallest step 2^-24 of a format in which the strong one is 1, and together
    they are the result. The kernels scale the weights by 2^15, or (packed, whose reference may lie
    2^8 below the maximum) by 2^7 at least: steps of 2^-31, each weight off by half of one."""
    at = {"first": 0, "middle": n // 2, "last": n - 1}[strong]
    q, k, v = (torch.zeros(r, 2, dim, device=DEV, dtype=torch.float16) for r in (1, n, n))
    q[0, :, 5], k[:, :, 5], v[:] = 1.0, -gap, 1.0
    k[at, :, 5], v[at] = 0.0, 0.0
    weak = (n - 1) * math.exp(-gap)
    want = torch.full((2, dim), weak / (1 + weak), device=DEV, dtype=torch.float64)
    u = 2.0 ** -11
    tol = (2 * u + 2.0 ** -16) * want + n * 2.0 ** -32 + 2.0 ** -25
    for name, out, lse in every_form(q, k, v, 1.0):
        check(out, want, tol, name)
        check(lse, torch.full((2,), math.log1p(weak), device=DEV, dtype=torch.float64), torch.full((2,), n * 2.0 ** -24 + 2.0 ** -20, device=DEV, dtype=torch.float64), name + ", log-sum")


# ---- arguments -------------------------------------------------------------------------------
def refused(call, text):
    with pytest.raises(dv.DINOv3Error) as e:
        call()
    assert e.value.code == dv.INVALID_ARGUMENT and text in str(e.value), str(e.value)


def test_caches_without_slots_are_refused():
    q, none = torch.zeros(2, 4, 64, device=DEV, dtype=torch.float16), torch.empty(3, 4, 0, 64, device=DEV, dtype=torch.float16)
    table, n = ints([[0, 1], [2, 0]]), ints([1, 1])
    refused(lambda: dv.attention_paged(q, none, none, table, n), "page_size")
    refused(lambda: dv.attention_paged(q, none, none, table, n, workspace=torch.empty(1 << 20, dtype=torch.uint8, device=DEV)), "page_size")
    refused(lambda: dv.rope_append(q, q, q, none, none, table, n), "page_size")


def test_outputs_beside_inputs_in_one_buffer():
    """Views that share a buffer but no element are taken; those that share one are refused and leave
    the buffer as it was."""
    g, t, dim, cu = gen(83), 150, 64, ints([0, 100, 150])
    qkv = randn(g, t, 12, dim, dtype=torch.float16)  # 4 query, 2 key, 2 value heads, 4 of the result
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:8]
    want = dv.attention_packed(q, k, v, cu, causal=True)
    dv.attention_packed(q, k, v, cu, causal=True, out=qkv[:, 8:])
    assert torch.equal(qkv[:, 8:], want)
    heads = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    dv.attention_packed(heads[:, :4], heads[:, 4:6], heads[:, 6:8], cu, causal=True, out=heads[:, 8:])
    assert torch.equal(heads[:, 8:], want)
    both_rows = torch.cat([qkv[:, :4], torch.zeros_like(qkv[:, :4])])  # queries, then results
    dv.attention_packed(both_rows[:t], k, v, cu, causal=True, out=both_rows[t:])
    assert torch.equal(both_rows[t:], want)
    before = qkv.clone()
    for out in (qkv[:, 1:5], qkv[:, 7:11], qkv[:, 4:8], q):
        refused(lambda: dv.attention_packed(q, k, v, cu, out=out), "overlap")
    refused(lambda: dv.attention_packed(both_rows[:t], k, v, cu, out=both_rows[t - 1:-1]), "overlap")
    assert torch.equal(qkv, before)

    pool, lens, table = torch.zeros(12, 2, 2, 16, dim, device=DEV, dtype=torch.float16), ints([100, 50]), ints([[0, 1, 2, 3, 4, 5, 6], [7, 8, 9, 10, -1, -1, -1]])
    kc, vc = pool[:, 0], pool[:, 1]
    cos = torch.rand(128, 32, device=DEV)
    apart_q = dv.rope_append(q, k, v, kc, vc, table, lens, cos, cos, cu_new=cu)
    again, kept = qkv.clone(), pool.clone()
    mine = again[:, :4]  # in place within the fused rows
    assert dv.rope_append(mine, again[:, 4:6], again[:, 6:8], kc, vc, table, lens, cos, cos, cu_new=cu, q_out=mine) is mine
    assert torch.equal(mine, apart_q) and torch.equal(again[:, 4:], qkv[:, 4:]) and torch.equal(pool, kept)
    refused(lambda: dv.rope_append(q, k, v, kc, vc, table, lens, cos, cos, cu_new=cu, q_out=qkv[:, 1:5]), "overlap")
    refused(lambda: dv.rope_append(q, k, v, kc, kc, table, lens, cos, cos, cu_new=cu), "overlap")
    rows = pool[0].view(-1, 2, dim)[:2]  # two rows inside the first page
    refused(lambda: dv.rope_append(None, rows, rows, kc, vc, table, ints([1, 1])), "overlap")
    refused(lambda: dv.attention_paged(q[:2], kc, vc, table, lens, out=pool[3].view(-1, 4, dim)[:2]), "overlap")
    assert torch.equal(qkv, before) and torch.equal(pool, kept)


# ---- gradients -------------------------------------------------------------------------------
def everything(dtype=torch.float16):
    """The float tensors of a call of each operator by name, and the calls on such a dict."""
    g = gen(84)
    t = {n: randn(g, 6, h, 64, dtype=dtype) for n, h in (("q", 4), ("k", 2), ("v", 2), ("out", 4))}
    t.update({n: torch.zeros(3, 2, 8, 64, device=DEV, dtype=dtype) for n in ("k_cache", "v_cache")})
    t.update(cos=torch.rand(16, 32, device=DEV), sin=torch.rand(16, 32, device=DEV), lse=torch.zeros(6, 4, device=DEV))
    cu, table, lens, few = ints([0, 6]), ints([[0, 1]]), ints([6]), ints([[0, 1]] * 6)
    calls = {
        "packed": (("q", "k", "v", "out", "lse"), lambda t: dv.attention_packed(t["q"], t["k"], t["v"], cu, out=t["out"], lse=t["lse"])),
        "append": (("q", "k", "v", "out", "k_cache", "v_cache", "cos", "sin"),
                   lambda t: dv.rope_append(t["q"], t["k"], t["v"], t["k_cache"], t["v_cache"], table, lens, t["cos"], t["sin"], cu_new=cu, q_out=t["out"])),
        "paged": (("q", "k_cache", "v_cache", "out", "lse"), lambda t: dv.attention_paged(t["q"], t["k_cache"], t["v_cache"], few, ints([6] * 6), out=t["out"], lse=t["lse"])),
    }
    return t, calls


@pytest.mark.parametrize("op", ["packed", "append", "paged"])
def test_tensors_that_want_a_gradient(op):
    tensors, calls = everything()
    names, call = calls[op]
    call(tensors)
    for name in names:
        wanting = dict(tensors, **{name: tensors[name].clone().requires_grad_()})
        refused(lambda: call(wanting), "requires a gradient")
        with torch.no_grad():
            call(wanting)


@pytest.mark.parametrize("op", ["packed", "append", "paged"])
def test_tensors_that_carry_a_tangent(op):
    """Forward-mode dual tensors, whose tangent the result would not have; under no_grad as well, which
    does not switch forward mode off."""
    from torch.autograd import forward_ad

    tensors, calls = everything()
    names, call = calls[op]
    for name in names:
        with forward_ad.dual_level():
            dual = dict(tensors, **{name: forward_ad.make_dual(tensors[name].clone(), torch.ones_like(tensors[name]))})
            refused(lambda: call(dual), "tangent")
            with torch.no_grad():
                refused(lambda: call(dual), "tangent")
    call(tensors)


def test_what_a_call_writes_counts_as_changed():
    """A tensor that autograd keeps for a backward pass and a call overwrites meanwhile is noticed, as
    torch's own operators in place are; inference tensors, which have no counter, are written."""
    tensors, calls = everything(torch.bfloat16)
    written = {"packed": ("out", "lse"), "append": ("out", "k_cache", "v_cache"), "paged": ("out", "lse")}
    for op, (names, call) in calls.items():
        before = {n: tensors[n]._version for n in names}
        call(tensors)
        assert {n for n in names if tensors[n]._version != before[n]} == set(written[op]), op
        call({n: x.detach() for n, x in tensors.items()})
        with torch.inference_mode():
            held = {n: x.clone() for n, x in tensors.items()}
            call(held)
        call(held)
    weight = torch.ones(64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    loss = (tensors["k_cache"] * weight).sum()
    calls["append"][1](tensors)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_an_output_for_queries_that_are_not_given():
    tensors, _ = everything()
    refused(lambda: dv.rope_append(None, tensors["k"][:1], tensors["v"][:1], tensors["k_cache"], tensors["v_cache"], ints([[0, 1]]), ints([1]), q_out=tensors["out"][:1]),
            "q_out goes with q")


# ---- workspaces ------------------------------------------------------------------------------
def test_one_workspace_for_calls_of_any_length():
    """Calls from one token to a long split in one workspace of the bounding size, as without one."""
    g, hq, hkv, dim = gen(85), 8, 2, 64
    paged = torch.full((dv.attention_paged_workspace(40, hq, hkv, dim),), 255, dtype=torch.uint8, device=DEV)
    packed = torch.full((dv.attention_packed_workspace(dim, DEV),), 255, dtype=torch.uint8, device=DEV)
    for lens in ([1], [300], [70, 5000], [8, 0, 900] * 10, [2000] * 40, [20000]):
        k, v, table = paged_cache(86, lens, hkv, 16, dim, torch.float16)
        q = randn(g, len(lens), hq, dim, dtype=torch.float16)
        for max_len in (None, 64, max(lens)):
            want = dv.attention_paged(q, k, v, table, ints(lens), max_len=max_len)
            assert torch.equal(want, dv.attention_paged(q, k, v, table, ints(lens), max_len=max_len, workspace=paged))
        k, v = randn(g, sum(lens), hkv, dim, dtype=torch.float16), randn(g, sum(lens), hkv, dim, dtype=torch.float16)
        cu = cu_of([1] * len(lens))
        want = dv.attention_packed(q, k, v, cu, cu_of(lens), causal=True)
        assert torch.equal(want, dv.attention_packed(q, k, v, cu, cu_of(lens), causal=True, workspace=packed))
    for call in (lambda: dv.attention_packed_workspace(96), lambda: dv.attention_paged_workspace(4, 6, 4, 64), lambda: dv.attention_paged_workspace(0, 4, 4, 64)):
        refused(call, "no call has")


# ---- many sequences --------------------------------------------------------------------------
def shortest(call):
    """Milliseconds of the quickest of four calls, the host's pauses left out by that."""
    times = []
    for _ in range(4):
        marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        marks[0].record()
        call()
        marks[1].record()
        torch.cuda.synchronize()
        times.append(marks[0].elapsed_time(marks[1]))
    return min(times)


def test_append_between_many_empty_sequences():
    """Rows of one warp whose sequences lie a million empty ones apart. Each is found in some twenty steps; a
    walk over the empty ones took 0.19 s, so 50 ms tell the two apart."""
    n, rows = 3_000_000, 3
    at = [5, 1_000_000, n - 7]  # the sequences with a row
    ends = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    for s in at:
        ends[s + 1:] += 1
    lens = torch.zeros(n, dtype=torch.int32, device=DEV)
    lens[at] = ints([1, 2, 3])
    table = torch.full((n, 1), -1, dtype=torch.int32, device=DEV)
    table[at, 0] = ints([2, 0, 1])
    k_cache, v_cache = (torch.zeros(3, 1, 16, 64, device=DEV, dtype=torch.float16) for _ in range(2))
    k, v = randn(gen(87), rows, 1, 64, dtype=torch.float16), randn(gen(88), rows, 1, 64, dtype=torch.float16)
    took = shortest(lambda: dv.rope_append(None, k, v, k_cache, v_cache, table, lens, cu_new=ends))
    for row, (page, slot) in enumerate(((2, 0), (0, 1), (1, 2))):
        assert torch.equal(k_cache[page, 0, slot], k[row, 0]) and torch.equal(v_cache[page, 0, slot], v[row, 0])
    assert k_cache.count_nonzero() <= rows * 64 and took < 50


@pytest.mark.parametrize("hq,hkv,dim", [(32, 8, 128), (8, 2, 64), (33, 1, 64)])
@pytest.mark.parametrize("active,length", [(1, 4000), (3, 200), (5, 900), (0, 0)])
def test_paged_slots_that_are_empty(active, length, hq, hkv, dim):
    """A batch of fixed size, most of whose sequences have no tokens, as a captured decoder's step has it: the
    values, the empty ones' zeros, and the time. Each empty unit took a warp 1 us, one behind the other: 38 ms
    for 4096 slots and one of 4000 tokens. Its zeros are 32 MB, 5 us: 3 ms tell the two apart."""
    slots = 4096
    at = sorted({(i * 1237 + 7) % slots for i in range(active)} | ({slots - 1} if active > 1 else set()))
    lens = [0] * slots
    for i in at:
        lens[i] = length
    k, v, table = paged_cache(89, lens, hkv, 16, dim, torch.bfloat16, wide=256)
    q = randn(gen(90), slots, hq, dim, dtype=torch.bfloat16)
    n = ints(lens)
    none = n == 0
    for max_len in (None, max(length, 1)):
        out, lse = torch.full_like(q, 3.0), torch.full((slots, hq), 3.0, device=DEV)
        took = shortest(lambda: dv.attention_paged(q, k, v, table, n, max_len=max_len, out=out, lse=lse))
        assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
        assert took < 3
        for i in at:
            o, tol, l, ltol = one_sequence(q[i:i + 1], cached_rows(k, table, i, length), cached_rows(v, table, i, length), dim ** -0.5, False)
            check(out[i:i + 1], o, tol, f"slot {i}")
            check(lse[i:i + 1], l, ltol, f"log-sum of slot {i}")
