"""The token-step operators where sizes, lengths and values run out: empty batches, bad lengths, the ends of number ranges."""
import numpy as np
import pytest

import tadma_b200 as tb
from tadma_b200.abi import Status
from tests import token_step_reference as ref
from tests.token_step_reference import UNIT, f64

pytestmark = pytest.mark.gpu

INDEX = 1 << Status.ERR_INDEX


def torch_():
    import torch
    return torch


def gen(seed):
    return torch_().Generator(device="cuda").manual_seed(seed)


def ints(v, dtype="int32"):
    torch = torch_()
    return torch.tensor(np.asarray(v), dtype=getattr(torch, dtype), device="cuda")


@pytest.fixture(autouse=True)
def _clean_flags():
    tb.error_flags()
    yield
    tb.error_flags()


# ------------------------------------------------------------ block tables --

@pytest.mark.parametrize("slots_type", ["int32", "int64"])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("cap", [0, 5, 3000])
def test_block_tables_of_an_empty_batch(slots_type, strided, cap):
    torch = torch_()
    step = 3 if strided else 1

    def out(n, dtype="int32"):
        return torch.full((n * step,), 99, dtype=getattr(torch, dtype), device="cuda")[::step]

    def call(held, added, left_in, slots, width):
        n = len(held)
        table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        starts, lens, left = out(n + 1), out(n), out(1)
        tb.block_tables(ints(held), ints(added), torch.arange(20000, dtype=torch.int32, device="cuda"), ints([left_in]), 16, table, slots,
                        starts, lens, left)
        return starts, left

    # a large batch first: its sums are what shared memory is left with
    call([40] * 1000, [300] * 1000, 20000, out(300000), 30)
    assert tb.error_flags() == 0
    slots = out(cap, slots_type)
    starts, left = call([], [], 11, slots, 30)
    assert tb.error_flags() == 0
    assert starts.tolist() == [0] and left.tolist() == [11] and bool((slots == -1).all())


def one_request(held, added, page_size, entries, slots_type="int64"):
    """(slots, flags) of one request with that table row and an empty pool."""
    torch = torch_()
    slots, starts, lens, left = (torch.full((k,), 99, dtype=getattr(torch, t), device="cuda")
                                 for k, t in ((added, slots_type), (2, "int32"), (1, "int32"), (1, "int32")))
    tb.block_tables(ints([held]), ints([added]), ints([0]), ints([0]), page_size, ints([entries]), slots, starts, lens, left)
    return slots.tolist(), tb.error_flags()


def test_block_tables_flags_slots_that_int32_cannot_hold():
    page_size = 1 << 20
    at = 2 ** 31 - 2  # of page 2047 the last place but one
    assert one_request(at % page_size, 2, page_size, [2047], "int32") == ([at, at + 1], 0)
    assert one_request(5, 2, page_size, [2048], "int64") == ([2 ** 31 + 5, 2 ** 31 + 6], 0)
    assert one_request(5, 2, page_size, [2048], "int32") == ([-1, -1], INDEX)


def test_block_tables_flags_tokens_past_the_width():
    # the last held page is half full, so no new page is needed, but the table has no entry for it
    assert one_request(20, 3, 16, [4]) == ([-1] * 3, INDEX)
    assert one_request(20, 3, 16, [4, 7]) == ([116, 117, 118], 0)
    assert one_request(20, 3, 16, [4, -1]) == ([-1] * 3, 0)  # an entry without a page is the caller's


# -------------------------------------------------------------- the cache --

@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128), (256, 64)])
def test_append_of_equal_slots_changes_no_other(dim, group):
    # 600 tokens on 40 slots.  Where all tokens of a slot are the same it holds them; what the others hold is not defined.
    torch = torch_()
    g = gen(dim)
    tokens, heads, page = 600, 2, 16
    slots = torch.arange(tokens, device="cuda") % 40 + 17
    x = [torch.randn((tokens, heads, dim), device="cuda", generator=g).half() for _ in range(2)]
    same = slots % 2 == 0
    for t in x:
        t[same] = t[slots[same] - 17]
    shape = (8, heads, page)
    caches = [(torch.randint(0, 256, shape + (dim // 2,), dtype=torch.uint8, device="cuda", generator=g),
               torch.randn(shape + (dim // group, 2), device="cuda", generator=g).half()) for _ in range(2)]
    before = [[t.clone() for t in c] for c in caches]
    tb.kv4_append(*x, slots, *caches[0], *caches[1])
    assert tb.error_flags() == 0
    others = np.setdiff1d(np.arange(8 * page), slots.cpu().numpy())
    even = slots[same].unique().cpu().numpy()
    for i in range(2):
        for now, was in zip(cache_rows(*caches[i], others), cache_rows(*before[i], others)):
            assert np.array_equal(now, was)
        alone = [torch.zeros_like(t) for t in caches[i]]
        tb.kv4_append(x[i][:40], x[i][:40], slots[:40], *alone, *alone)
        for now, want in zip(cache_rows(*caches[i], even), cache_rows(*alone, even)):
            assert np.array_equal(now, want)


# ------------------------------------------------------------------ logits --

@pytest.mark.parametrize("room", [4, 7, 8, 9000])
@pytest.mark.parametrize("at", [8, 9])  # ids on 16-byte boundaries, and off them
@pytest.mark.parametrize("bad", [[-1, -5], [-4, -1 << 31], [-3, -2]])
def test_logits_negative_lengths_are_empty(room, at, bad):
    torch = torch_()
    store = torch.arange(at + 3 * room + 8, dtype=torch.int32, device="cuda") % 50  # tokens before, between and behind the rows
    ids = store[at:at + 3 * room].view(3, room)
    x = torch.ones((3, 50), device="cuda")
    out = torch.zeros_like(x)
    two = torch.full((3,), 2.0, device="cuda")
    tb.adjust_logits(x, ids, ints([room, 0, 0]), ints(bad + [2]), out, repetition=two, presence=two, frequency=two)
    assert tb.error_flags() & INDEX
    want = torch.ones_like(x)
    for t in ids[2, :2].tolist():
        want[2, t] = 0.5 - 2.0 - 2.0
    assert torch.equal(out, want)


# --------------------------------------------------------------- attention --

def test_attention_of_more_tokens_than_an_int_counts():
    # One page of 2^20 tokens, 2048 times in a table: a length of 2^31 - 1 is cut to 2^31 - 64 and flagged.  The result
    # is that of the page alone, but for the rounding of long sums: a warp has at least 2^31 / (148 * 16) tokens, which
    # at two additions a 32 tokens, each within 2^-23 of the sum, are 56,680 of them: 2^-7.2 of the weighted magnitude
    # at the very most, and the weights' own sum half of that.
    torch = torch_()
    g = gen(11)
    page, dim = 1 << 20, 64
    codes = torch.randint(0, 256, (1, 1, page, dim // 2), dtype=torch.uint8, device="cuda", generator=g)
    params = torch.tensor([0.25, -1.5], device="cuda").half().expand(1, 1, page, 1, 2).contiguous()
    q = torch.randn((1, 1, dim), device="cuda", generator=g).half()
    table = torch.zeros((1, 2048), dtype=torch.int32, device="cuda")
    one, all_ = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    tb.kv4_attention(q, codes, params, codes, params, table, ints([page]), 0.125, one)
    assert tb.error_flags() == 0
    tb.kv4_attention(q, codes, params, codes, params, table, ints([2 ** 31 - 1]), 0.125, all_)
    assert tb.error_flags() & INDEX
    assert float((one.float() - all_.float()).abs().max()) <= 2.0 ** -6 * 2.25 + 2.0 ** -10  # |values| are at most 2.25


def cache_rows(codes, params, slots):
    """Host rows [tokens, heads, ...] of a cache at those slots."""
    page = codes.shape[2]
    return [t.cpu().numpy()[slots // page, :, slots % page] for t in (codes, params)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 64), (128, 128), (256, 32), (256, 256)])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 1)])
@pytest.mark.parametrize("spare", [0, 3000])
def test_attention_scores_of_queries_with_a_mean(dtype, dim, group, heads, kv_heads, spare):
    # Keys (c - 8) s with c = 8 but in 8 of their places, queries of about 4 everywhere: what the scores are made of is
    # small beside any multiple of sum q.  A step of mma.sync adds 17 terms, aligned to the largest and cut to 24 bits or
    # more: 17 * 2^-24 < 2^-19.9 of the largest, which is at most A = sum |q||k|.  So a score errs by less than
    # (dim / 16 + 4) 2^-19.9 A scale, a weight by twice the largest of these and 2^-17 for the exponential and the two
    # halves of p s, and the values' sum by as much a step again: two steps (with the halves apart) a 16 tokens.
    torch = torch_()
    g = gen(dim + group + heads)
    lens, page, scale = [300, 77], 16, 0.25
    params, codes = [], []
    for i in range(2):
        s = 2.0 ** torch.randint(-1, 2, (26, kv_heads, page, dim // group, 1), device="cuda", generator=g)
        params.append(torch.cat([s, -8 * s], -1).half())
        nibbles = torch.full((26, kv_heads, page, dim), 8, dtype=torch.uint8, device="cuda")
        at = torch.rand(nibbles.shape, device="cuda", generator=g).argsort(-1)[..., :8]
        nibbles.scatter_(-1, at, torch.randint(7, 10, at.shape, dtype=torch.uint8, device="cuda", generator=g))
        if i == 1:
            nibbles = torch.randint(0, 16, nibbles.shape, dtype=torch.uint8, device="cuda", generator=g)
        codes.append(nibbles[..., 0::2] | nibbles[..., 1::2] << 4)
    table = torch.randperm(26, device="cuda", generator=g).int()[None].repeat(2, 1)
    table = torch.cat([table, torch.full((2, spare), -1, dtype=torch.int32, device="cuda")], 1)
    q = (4 + 0.5 * torch.randn((2, heads, dim), device="cuda", generator=g)).clamp(min=1).to(getattr(torch, dtype))
    out = torch.full_like(q, 7.0)
    tb.kv4_attention(q, codes[0], params[0], codes[1], params[1], table, ints(lens), scale, out)
    assert tb.error_flags() == 0
    got, qh, tab = f64(out), f64(q), table.cpu().numpy()
    for r, n in enumerate(lens):
        t = np.arange(n)
        slots = tab[r][t // page].astype(np.int64) * page + t % page
        kk, vv = (ref.values(*cache_rows(c, p, slots)) for c, p in zip(codes, params))
        want, mass, top = ref.attention(qh[r], kk, vv, scale)
        step = 17 * 2.0 ** -24
        weight = 2 * (dim / 16 + 4) * step * top[:, None] + 2.0 ** -17
        tol = UNIT[dtype] * np.abs(want) + (weight + (n / 8 + 4) * step) * (mass + np.abs(want))
        off = np.abs(got[r] - want)
        assert np.all(off <= tol), (r, float((off / tol).max()), float(off.max()))


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1)])
@pytest.mark.parametrize("requests,n", [(1, 4096), (200, 352)])
@pytest.mark.parametrize("first,ahead,rest", [(0.0, 8.0, 1e-3), (64.0, -40.0, 2.0 ** -20), (2.0 ** -20, -40.0, 64.0)])
@pytest.mark.parametrize("spread", [False, True])  # scores that differ from token to token
def test_attention_of_value_scales_far_apart(heads, kv_heads, requests, n, first, ahead, rest, spread):
    # Every fourth tile of 32 tokens has value scales of another size and scores `ahead` of the others', so that a
    # running scaling of the weights has to follow.  Products p s keep 2^-18 of themselves and sums some 2^-20 a step
    # (n / 8 steps at most), well inside 2^-9; results are rounded to bfloat16.
    torch = torch_()
    g = gen(requests + heads)
    dim, page = 64, 16
    pages = requests * n // page
    tiles = (torch.arange(n, device="cuda") // 32 % 4 == 0).view(1, n // page, 1, page)

    def per_token(there, elsewhere):
        t = torch.where(tiles, float(there), float(elsewhere)).expand(requests, n // page, kv_heads, page)
        return t.reshape(pages, kv_heads, page, 1)

    zero = torch.zeros((pages, kv_heads, page, 1), device="cuda")
    k = [torch.zeros((pages, kv_heads, page, dim // 2), dtype=torch.uint8, device="cuda"),
         torch.stack([zero, per_token(ahead / 8, 0)], -1).half()]
    if spread:
        k[0].random_(0, 256, generator=g)
        k[1][..., 0] = 0.125
    v = [torch.randint(0, 4, (pages, kv_heads, page, dim), dtype=torch.uint8, device="cuda", generator=g) + 12,
         torch.stack([per_token(first, rest), zero], -1).half()]
    v[0] = v[0][..., 0::2] | v[0][..., 1::2] << 4
    q = torch.ones((requests, heads, dim), dtype=torch.bfloat16, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(requests, -1)
    out = torch.full_like(q, 7.0)
    tb.kv4_attention(q, *k, *v, table, ints([n] * requests), 0.125, out)  # scores are 8 times the keys' value
    assert tb.error_flags() == 0
    got = f64(out)
    for r in range(0, requests, 7):
        slots = np.arange(r * n, (r + 1) * n)
        kk, vv = (ref.values(*cache_rows(*c, slots)) for c in (k, v))
        want, mass, _ = ref.attention(np.ones((heads, dim)), kk, vv, 0.125)
        off = np.abs(got[r] - want)
        tol = UNIT["bfloat16"] * np.abs(want) + 2.0 ** -9 * mass
        assert np.all(off <= tol), (r, float((off / tol).max()))


@pytest.mark.parametrize("size,scale", [(2.0 ** -100, 0.0), (2.0 ** -60, 0.0), (1.0, 0.0), (2.0 ** 110, 0.0), (2.0 ** -110, 1e-12), (2.0 ** -90, -1e-20),
                                        (2.0 ** -100, 2.0 ** 97), (2.0 ** 100, -(2.0 ** -103))])
@pytest.mark.parametrize("spare", [0, 3000])
def test_attention_of_tiny_and_huge_queries(size, scale, spare):
    # bfloat16 queries of any magnitude.  A score errs by 2^-16 of sum |q||k| scale and a weight by 2^-13, as bounded for
    # ordinary queries; sizes are powers of two.
    torch = torch_()
    g = gen(21)
    lens, heads, dim, page = [77, 40, 1], 4, 64, 16
    pages = 12
    caches = []
    for _ in range(2):
        s = torch.rand((pages, 2, page, 2, 1), device="cuda", generator=g) * 0.3 + 0.1
        caches.append((torch.randint(0, 256, (pages, 2, page, dim // 2), dtype=torch.uint8, device="cuda", generator=g),
                       torch.cat([s, -7.5 * s], -1).half()))
    table = torch.cat([torch.arange(15, device="cuda").view(3, 5).int() % pages, torch.full((3, spare), -1, dtype=torch.int32, device="cuda")], 1)
    q = (torch.randn((3, heads, dim), device="cuda", generator=g).bfloat16().double() * size).bfloat16()
    out = torch.full_like(q, 7.0)
    tb.kv4_attention(q, *caches[0], *caches[1], table, ints(lens), scale, out)
    assert tb.error_flags() == 0
    got, tab = f64(out), table.cpu().numpy()
    for r, n in enumerate(lens):
        t = np.arange(n)
        slots = tab[r][t // page].astype(np.int64) * page + t % page
        kk, vv = (ref.values(*cache_rows(*c, slots)) for c in caches)
        want, mass, top = ref.attention(f64(q)[r], kk, vv, scale)
        tol = UNIT["bfloat16"] * np.abs(want) + (2.0 ** -13 + 2.0 ** -16 * top[:, None]) * (mass + np.abs(want))
        off = np.abs(got[r] - want)
        assert np.all(off <= tol), (r, float(np.nanmax(off / tol)))


# ------------------------------------------------------------------ matvec --

@pytest.mark.parametrize("dtype,size", [("float16", 1.0), ("bfloat16", 1.0), ("bfloat16", 2.0 ** 118), ("bfloat16", 2.0 ** 125)])
@pytest.mark.parametrize("m", [1, 5, 12])
@pytest.mark.parametrize("n,k,group,zeros", [(5, 64, 32, True), (100, 640, 64, False), (300, 8192, 128, True), (6000, 2112, 32, True)])
def test_matvec_of_infinite_and_huge_rows(dtype, size, m, n, k, group, zeros):
    # Row 0 has an infinity, row 1 two of them, row 2 a NaN; the others are numbers, of the end of bfloat16's range
    # (scales keep the results inside fp32's).  A result is an infinity or NaN where the formula gives one; numbers err by a
    # rounding a term of 32, one a block of 32, and that of the fast form, 2^-18 of sum |x| 16 s.
    torch = torch_()
    g = gen(m + n + k)
    x = (torch.randn((m, k), device="cuda", generator=g).clamp(-4, 4) * size).to(getattr(torch, dtype))
    x[0, k // 3] = float("inf")
    if m > 2:
        x[1, 7], x[1, k - 1] = float("-inf"), float("inf")
        x[2, k // 2] = float("nan")
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = ((torch.rand((n, k // group), device="cuda", generator=g) + 0.5) * 2.0 ** -13).to(getattr(torch, dtype))
    z = torch.randint(0, 16, (n, k // group), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    bias = torch.randn(n, device="cuda", generator=g)
    out = torch.full((m, n), 7.0, device="cuda")
    tb.matvec_q4(x, codes, scales, out, zeros=z, bias=bias)
    w = ref.weights(codes.cpu().numpy(), f64(scales), None if z is None else z.cpu().numpy())
    xh, got = f64(x), f64(out)
    plain = np.where(np.isfinite(xh), xh, 0.0)
    want, size_of = plain @ w.T + f64(bias), np.abs(plain) @ np.abs(w).T
    fast = np.abs(plain) @ np.repeat(16 * f64(scales), group, 1).T
    with np.errstate(invalid="ignore"):
        for r in range(min(m, 3)):
            for at in np.flatnonzero(~np.isfinite(xh[r])):
                want[r] += xh[r, at] * w[:, at]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    finite = np.isfinite(want)
    tol = UNIT["float32"] * np.abs(want) + (33 + k / 32) * 2.0 ** -24 * size_of + 2.0 ** -18 * fast
    assert np.all(np.abs(got[finite] - want[finite]) <= tol[finite])


# ----------------------------------------------------------------- threads --

def in_threads(*calls, times=4000):
    """Runs the calls `times` times each, every one in a thread and on a stream of its own; raises what one raises."""
    import threading
    torch = torch_()
    errors, gate = [], threading.Barrier(len(calls))

    def work(call, stream):
        gate.wait()
        try:
            for _ in range(times):
                call(stream)
        except Exception as e:  # noqa: BLE001  (handed to the test)
            errors.append(e)

    streams = [torch.cuda.Stream() for _ in calls]
    threads = [threading.Thread(target=work, args=(c, s.cuda_stream)) for c, s in zip(calls, streams)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    if errors:
        raise errors[0]


def test_matvec_of_few_and_more_rows_in_two_threads():
    # One kernel, 51,200 bytes of shared memory a CTA for 2 rows and 100,352 for 8.
    torch = torch_()
    g = gen(31)
    n, k = 256, 512
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.full((n, k // 128), 0.01, dtype=torch.float16, device="cuda")
    xs = [torch.randn((m, k), device="cuda", generator=g).half() for m in (2, 8)]
    outs = [torch.zeros((x.shape[0], n), dtype=torch.float32, device="cuda") for x in xs]
    in_threads(*[lambda stream, x=x, out=out: tb.matvec_q4(x, codes, scales, out, stream=stream) for x, out in zip(xs, outs)])
    for x, out in zip(xs, outs):
        alone = torch.zeros_like(out)
        tb.matvec_q4(x, codes, scales, alone)
        assert torch.equal(out, alone)


def test_block_tables_of_many_and_more_requests_in_two_threads():
    # 12 bytes of shared memory a request: 60,008 for 5000 and 192,008 for 16000.
    torch = torch_()

    def make(n):
        held, added = ints([17] * n), ints([1] * n)
        table = torch.zeros((n, 2), dtype=torch.int32, device="cuda")
        out = [torch.full((k,), 99, dtype=torch.int32, device="cuda") for k in (n, n + 1, n, 1)]
        args = [held, added, ints([0]), ints([1]), 16, table, *out]
        return lambda stream: tb.block_tables(*args, stream=stream), out

    (few, few_out), (more, more_out) = make(5000), make(16000)
    in_threads(few, more)
    assert tb.error_flags() == 0
    for n, (slots, starts, lens, left) in ((5000, few_out), (16000, more_out)):
        assert bool((slots == 1).all()) and torch.equal(starts, torch.arange(n + 1, dtype=torch.int32, device="cuda"))
        assert bool((lens == 18).all()) and left.tolist() == [1]


# -------------------------------------------------------------- error word --

def in_a_process(program):
    """What a Python program prints that runs in a process of its own."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_error_flags_copies_one_word():
    # whatever operator set it: reading is one copy from the device, clearing one to it (a profiler that another test
    # started and ended may record nothing in this process)
    copies = in_a_process("""
import torch, tadma_b200 as tb
x = torch.ones((1, 8), device="cuda")
tb.gather(x, 0, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty_like(x))
tb.error_flags()
with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU, torch.profiler.ProfilerActivity.CUDA]) as prof:
    assert tb.error_flags(clear=False) == 0
    assert tb.error_flags(clear=True) == 0
print(sorted(e.name.split()[1] for e in prof.events() if e.name.startswith("Memcpy")))
""")
    assert copies.strip() == "['DtoH', 'DtoH', 'HtoD']", copies


def test_error_word_is_one_for_all_operators():
    torch = torch_()
    x = torch.ones((1, 8), device="cuda")
    cache = [torch.zeros((1, 1, 16, 32), dtype=torch.uint8, device="cuda"), torch.zeros((1, 1, 16, 1, 2), dtype=torch.float16, device="cuda")]
    rows = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    spare = [ints([0] * n) for n in (2, 1, 1)]
    wrong = {"gather": lambda: tb.gather(x, 0, ints([5]), torch.empty_like(x)),
             "block_tables": lambda: tb.block_tables(ints([0]), ints([1]), ints([0]), ints([0]), 16, ints([[0]]), ints([0]), *spare),
             "kv4_append": lambda: tb.kv4_append(rows, rows, ints([16]), *cache, *cache),
             "kv4_read": lambda: tb.kv4_read(*cache, *cache, ints([-2]), rows.clone(), rows.clone()),
             "kv4_attention": lambda: tb.kv4_attention(rows, *cache, *cache, ints([[0]]), ints([17]), 0.125, rows.clone()),
             "adjust_logits": lambda: tb.adjust_logits(x, ints([[8]]), ints([0]), ints([1]), torch.empty_like(x))}
    for name, call in wrong.items():
        assert tb.error_flags() == 0, name
        call()
        assert tb.error_flags(clear=False) == INDEX, name
        assert tb.error_flags() == INDEX, name


def test_first_call_may_be_captured():
    # a process whose first calls of the library are recorded into a graph
    program = """
import torch, tadma_b200 as tb
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
x, out, ids, one = torch.ones((1, 8), device="cuda"), torch.zeros((1, 8), device="cuda"), i([[3, 9]]), i([2])
cache = [torch.zeros((1, 1, 16, 32), dtype=torch.uint8, device="cuda"), torch.zeros((1, 1, 16, 1, 2), dtype=torch.float16, device="cuda")]
rows, zero, pen = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda"), i([0]), torch.ones(1, device="cuda")
got, lens, table = rows.clone() + 1, i([1]), i([[0]])
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    tb.kv4_append(rows, rows, zero, *cache, *cache)
    tb.kv4_attention(rows, *cache, *cache, table, lens, 0.125, got)
    tb.adjust_logits(x, ids, zero, one, out, presence=pen)
g.replay()
torch.cuda.synchronize()
assert out.tolist() == [[1, 1, 1, 0, 1, 1, 1, 1]] and bool((got == 0).all()) and tb.error_flags() == 16
print("replayed")
"""
    assert "replayed" in in_a_process(program)
