"""The 8-bit key/value cache on a GPU against the 64-bit restatement in oracle/cache8.py: appending, attention, eviction, and a run of them."""
import math

import pytest
import torch

from oracle import cache8 as oc

pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    from teenygrad_b200 import ops
    assert ops.device_error() == 0


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def filled(seed, slots, kv, cap, dim, vdim, block, weights=False):
    """A cache of random codes (no NaN) under scales of several sizes, on the GPU, and its restatement."""
    from teenygrad_b200 import ops
    g = torch.Generator().manual_seed(seed)
    blocks = -(-cap // block)
    code = lambda d: oc.encode((torch.randn(slots, kv, cap, d, generator=g) * 90).clamp(-448, 448).double())  # noqa: E731
    scale = lambda: 2.0 ** torch.randint(-9, -5, (slots, kv, blocks), generator=g).float()  # noqa: E731
    k, v, ks, vs = code(dim), code(vdim), scale(), scale()
    w = torch.rand(slots, kv, cap, generator=g) if weights else None
    f8 = lambda t: t.cuda().view(torch.float8_e4m3fn)  # noqa: E731
    return ops.Cache8(f8(k), f8(v), ks.cuda(), vs.cuda(), block, None if w is None else w.cuda()), oc.Cache(k, v, ks, vs, block, w)


def same(cache, want, weights=True):
    """Every code (all NaN codes are one), scale and weight of the cache, written or not."""
    for got, codes in ((cache.k, want.k), (cache.v, want.v)):
        a, b = oc.VALUES[got.view(torch.uint8).cpu().long()], oc.VALUES[codes.long()]
        assert torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(b, nan=1e9))
    assert torch.equal(cache.k_scale.double().cpu(), want.ks) and torch.equal(cache.v_scale.double().cpu(), want.vs)
    if weights and want.weights is not None:
        assert torch.equal(torch.nan_to_num(cache.weights.double().cpu(), nan=-7.0), torch.nan_to_num(want.weights, nan=-7.0))


def rows_of(lens, slots, pos, gap=0):
    row, out = gap, []
    for n, s, p in zip(lens, slots, pos):
        out.append((s, p, row, n))
        row += n + gap
    return out, row


# ------------------------------------------------------------------------------------------------ append
@DTYPES
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,dim,vdim", [(2, 128, 128), (3, 64, 48), (1, 16, 80)])
def test_append(dtype, block, kv, dim, vdim):
    from teenygrad_b200 import ops
    cap = 300
    cache, want = filled(1, 5, kv, cap, dim, vdim, block, weights=True)
    # a whole prompt, a token in the middle of a block, one at a block's start, up to the last row, some over several blocks
    table, rows = rows_of([150, 1, 1, 44, 0, 2], [3, 0, 1, 2, 4, 4], [0, 77, 128, 256, 3, 127], gap=1)
    size = torch.exp(1.5 * rnd(2, rows, 1, 1))  # scales grow and stay
    k, v = (size * rnd(3, rows, kv, dim)).to(dtype), (size * rnd(4, rows, kv, vdim)).to(dtype)
    k[table[0][2] + 3, 0, :4] = torch.tensor([448.0, 1e-9, -0.0, 447.0]).to(dtype)
    ops.cache8_append(cache, k.cuda(), v.cuda(), ops.step_table(table))
    want.append(k, v, table)
    same(cache, want)


@DTYPES
def test_append_of_zeros_of_what_is_not_finite_and_of_extremes(dtype):
    from teenygrad_b200 import ops
    cache, want = filled(1, 2, 2, 64, 32, 16, 16)
    table, rows = rows_of([40, 20], [1, 0], [0, 9])
    k, v = rnd(3, rows, 2, 32).to(dtype), rnd(4, rows, 2, 16).to(dtype)
    inf = float("inf")
    k[3, 0, 2], k[4, 1, 3], k[5, 0, 0], v[41, 1, 1] = inf, -inf, float("nan"), inf
    k[16:32, 0], v[16:32] = 0.0, -0.0                                     # blocks of zeros
    k[16:32, 1], v[32:40, 0] = 1e-39, 3e38                                # (subnormal in both types), the largest
    k[32:40, 1] = float("nan")
    ops.cache8_append(cache, k.cuda(), v.cuda(), ops.step_table(table))
    want.append(k, v, table)
    same(cache, want)


@DTYPES
def test_append_token_by_token_and_again(dtype):
    """The same tokens one at a time: scales grow step by step, and a second pass over the last block's tokens finds the old scale kept."""
    from teenygrad_b200 import ops
    cache, want = filled(5, 1, 2, 50, 32, 32, 32)
    k = (torch.linspace(0.01, 30, 50)[:, None, None] * rnd(1, 50, 2, 32)).to(dtype)
    v = (torch.linspace(30, 0.01, 50)[:, None, None] * rnd(2, 50, 2, 32)).to(dtype)
    for t in list(range(50)) + [40, 41]:
        entry = [(0, t, 0, 1)]
        ops.cache8_append(cache, k[t:t + 1].cuda(), v[t:t + 1].cuda(), ops.step_table(entry))
        want.append(k[t:t + 1], v[t:t + 1], entry)
    same(cache, want)


@DTYPES
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_append_from_views(dtype, offset):
    """k and v inside the rows of a fused projection, also where its rows are not made of 16-byte pieces."""
    from teenygrad_b200 import ops
    cache, want = filled(1, 2, 2, 70, 48, 16, 64)
    rows, wide = 66, 2 * (48 + 16) + offset + 5
    x = rnd(2, rows, wide).to(dtype).cuda()
    k, v = x[:, offset:offset + 96].unflatten(1, (2, 48)), x[:, offset + 96:offset + 128].unflatten(1, (2, 16))
    table = [(1, 2, 0, 60), (0, 63, 61, 5)]
    ops.cache8_append(cache, k, v, ops.step_table(table))
    want.append(k.cpu(), v.cpu(), table)
    same(cache, want)


# ------------------------------------------------------------------------------------------------ attention
def bounds(dtype, want, q, dim, longest, softcap):
    """Per element, how far a right result can be: a score is off by its sum's roundings (one half step each of products and partial sums)
    and by its query's two-term form (2^-18 of the row's largest number), a soft cap by 2^-20 of the cap; a probability relatively by twice that, by
    its exponential (2^-21), by its row's sum and, before the values' product, by two E4M3 roundings (bf16: 2^-8; f32 has 24 bits); the output by a rounding."""
    out, lse, mass, dots = want
    u = 2.0 ** -24
    delta = (dim + 8) * u * dots + 2.0 ** -20 * softcap
    if dtype == BF:
        delta = delta + 2.0 ** -18 * dots.clamp(min=1.0) * math.sqrt(dim)
    delta = delta + u * lse.abs() * 4 + (longest + 64) * u
    p = 2 * delta + 2.0 ** -20
    step = 2.0 ** -8 if dtype == BF else u
    return step * out.abs() + ((2.0 ** -8 if dtype == BF else 2 * u) + p[..., None]) * mass * 1.02 + 1e-30, delta, p


def check(got, lse, want, dtype, q, dim, longest, softcap, table):
    near, delta, _ = bounds(dtype, want, q, dim, longest, softcap)
    for _, _, row, n in table:
        at = slice(row, row + n)
        worst = ((got[at].double().cpu() - want[0][at]).abs() / near[at])
        assert n == 0 or float(worst.max()) <= 1.0, float(worst.max())
        if lse is not None and n:
            assert float(((lse[at].double().cpu() - want[1][at]).abs() / delta[at]).max()) <= 1.0


SHAPES = [(4, 4, 128, 128, 64), (8, 2, 128, 128, 16), (6, 2, 64, 48, 32), (5, 1, 80, 16, 128), (16, 2, 96, 128, 32), (24, 2, 16, 32, 16)]


def attend(dtype, shape, lens, pos, cap, softcap=0.0, extras=False, decay=None, lse=True, seed=0, gap=0, scratch=None):
    from teenygrad_b200 import ops
    heads, kv, dim, vdim, block = shape
    slots = [(3 * i + 1) % len(lens) if len(lens) % 3 else len(lens) - 1 - i for i in range(len(lens))]
    cache, want = filled(seed, len(lens), kv, cap, dim, vdim, block, weights=decay is not None)
    table, rows = rows_of(lens, slots, pos, gap)
    q = (1.5 * rnd(seed + 1, rows, heads, dim)).to(dtype)
    sink, gate = (rnd(seed + 2, heads), rnd(seed + 3, rows, heads * vdim).to(dtype)) if extras else (None, None)
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    z = torch.full((rows, heads), 3.0, device="cuda") if lse else None
    out = torch.full((rows, heads, vdim), 5.0, dtype=dtype, device="cuda")
    ops.cache8_attention(q.cuda(), cache, dim ** -0.5, ops.step_table(table), softcap=softcap, sink=up(sink), gate=up(gate), weight_decay=decay,
                         lse=z, out=out, scratch=scratch)
    ref = want.attention(q, dim ** -0.5, table, softcap, sink, gate, decay)
    longest = max(p + n for p, n in zip(pos, lens))
    check(out, z, ref, dtype, q, dim, longest, softcap, table)
    mine = torch.zeros(rows, dtype=torch.bool)
    for _, _, row, n in table:
        mine[row:row + n] = True
    assert bool((out.cpu()[~mine] == 5.0).all()) and (z is None or bool((z.cpu()[~mine] == 3.0).all()))
    if decay is not None:
        _, _, p = bounds(dtype, ref, q, dim, longest, softcap)
        gotw = cache.weights.double().cpu()
        for slot, at, row, n in table:
            live = at + n if n else 0
            assert torch.equal(gotw[slot, :, live:], want.weights[slot, :, live:])
            near = (float(p[row:row + n].max()) if n else 0.0) + (n * heads // kv + 4) * 2.0 ** -24
            assert float(((gotw[slot, :, :live] - want.weights[slot, :, :live]).abs() - near * want.weights[slot, :, :live] - 1e-30).clamp(min=0).sum()) == 0.0
    same(cache, want, weights=False)
    return cache


@DTYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_single_tokens(dtype, shape):
    attend(dtype, shape, [1, 1, 1, 1, 1, 1, 1], [0, 1, 15, 63, 64, 200, 299], 300)


@DTYPES
@pytest.mark.parametrize("softcap,extras", [(0.0, True), (6.0, False), (30.0, True)])
@pytest.mark.parametrize("shape", SHAPES[1:4], ids=str)
def test_caps_sinks_and_gates(dtype, shape, softcap, extras):
    attend(dtype, shape, [1, 1, 3, 20], [0, 130, 61, 190], 210, softcap, extras, seed=3)


@DTYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_few_tokens(dtype, shape):
    attend(dtype, shape, [2, 5, 1, 0, 11], [0, 126, 70, 12, 189], 200, gap=1, seed=7)


@DTYPES
@pytest.mark.parametrize("decay", [0.0, 1.0, 0.75])
@pytest.mark.parametrize("lens,pos", [([1, 1, 1], [0, 140, 76]), ([3, 1, 0, 17], [5, 128, 3, 111])])
@pytest.mark.parametrize("shape", [SHAPES[1], SHAPES[2]], ids=str)
def test_weights_of_the_cached_tokens(dtype, decay, lens, pos, shape):
    attend(dtype, shape, lens, pos, 150, 0.0, True, decay, lse=False, seed=11)
    attend(dtype, shape, lens, pos, 150, 9.0, False, decay, lse=True, seed=12)


@DTYPES
@pytest.mark.parametrize("lens,pos", [([130], [0]), ([64, 129, 257], [0, 100, 3])])
def test_prompts(dtype, lens, pos):
    attend(dtype, (4, 2, 128, 128, 64), lens, pos, 270, decay=0.5, seed=21)
    attend(dtype, (4, 2, 64, 48, 16), lens, pos, 263, 12.0, True, seed=22)
    attend(dtype, (3, 1, 80, 96, 32), lens, pos, 263, seed=23)


@DTYPES
@pytest.mark.parametrize("lens,pos", [([1, 1], [30, 100]), ([4, 3], [28, 99]), ([140, 150], [0, 0])])
def test_what_is_not_visible_does_not_count(dtype, lens, pos):
    """NaN codes and scales behind the live rows, and NaN keys and values in an entry's later tokens, which its earlier ones do not see."""
    from teenygrad_b200 import ops
    heads, kv, dim, block, cap = 8, 2, 128, 16, 170
    cache, want = filled(31, 2, kv, cap, dim, dim, block, weights=True)
    table, rows = rows_of(lens, [1, 0], pos)
    q = rnd(32, rows, heads, dim).to(dtype)
    for slot, p, _, n in table:
        for codes, scales in ((want.k, want.ks), (want.v, want.vs)):
            codes[slot, :, p + n:] = 255
            scales[slot, :, -(-(p + n) // block):] = float("nan")
        cache.weights[slot, :, p + n:] = float("nan")
    last = table[0]
    if last[3] > 1:
        want.k[last[0], 0, last[1] + last[3] - 1, 5] = 127
        want.v[last[0], 1, last[1] + last[3] - 2, 9] = 127
        want.v[last[0], 1, last[1] + last[3] - 1, 70] = 255
    for got, src in ((cache.k, want.k), (cache.v, want.v)):
        got.view(torch.uint8).copy_(src)
    cache.k_scale.copy_(want.ks)
    cache.v_scale.copy_(want.vs)
    out = ops.cache8_attention(q.cuda(), cache, 0.1, ops.step_table(table), weight_decay=0.0)
    ref = want.attention(q, 0.1, table)
    nan = torch.isnan(ref[0])
    assert torch.equal(torch.isnan(out.cpu()), nan)
    if last[3] > 1:
        first = last[2] + last[3] - 2
        assert not bool(nan[:first].any()) and bool(nan[first, 4:, 9].all()) and bool(nan[first + 1, :4].all())
    fix = lambda t: torch.nan_to_num(t, nan=0.0)  # noqa: E731
    check(fix(out), None, tuple(fix(t) for t in ref), dtype, q, dim, 170, 0.0, table)
    gotw = cache.weights.cpu()
    for slot, p, _, n in table:
        assert bool(torch.isnan(gotw[slot, :, p + n:]).all()) and not bool(torch.isnan(gotw[slot, 1, :p + n]).any())


@DTYPES
def test_an_entry_that_does_not_fit_is_left_out(dtype):
    """A table that the device has moved on since: the host's checks are past, the kernels leave the entry out."""
    from teenygrad_b200 import ops
    cache, want = filled(41, 3, 2, 40, 64, 64, 16, weights=True)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.weights)]
    table = ops.step_table([(0, 3, 0, 1), (1, 3, 1, 1), (2, 30, 2, 1)])
    x = rnd(42, 3, 4, 64).to(dtype)
    for bad in ((0, 40, 0, 1), (3, 0, 0, 1), (-1, 0, 0, 1), (0, -1, 0, 1), (0, 3, 3, 1), (0, 3, 0, 2), (0, 2 ** 31 - 1, 0, 1), (0, 3, -1, 1), (0, 3, 0, -5)):
        table.seqs.copy_(torch.tensor([bad, bad, bad], dtype=torch.int32))
        ops.cache8_append(cache, x[:, :2].contiguous().cuda(), x[:, 2:].contiguous().cuda(), table)
        out = torch.full((3, 4, 64), 5.0, dtype=dtype, device="cuda")
        ops.cache8_attention(x.cuda(), cache, 0.1, table, weight_decay=0.5, out=out)
        assert bool((out == 5.0).all())
        if not 0 <= bad[0] < 3 or not 0 <= bad[1] <= 40:
            assert bool((ops.cache8_evict(cache, table, 4, 1) == -1).all())
        for t, b in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.weights), before):
            assert torch.equal(t, b), bad


@pytest.mark.parametrize("dtype,shape,lens,weights,want", [
    (BF, (8, 2, 128, 128, 64), [1, 1], False, {"cache8_attention_kernel"}),
    (BF, (8, 2, 128, 128, 64), [1, 1], True, {"cache8_attention_kernel", "cache8_weights_kernel"}),
    (F32, (8, 2, 64, 64, 64), [130, 1], True, {"cache8_attention_kernel", "cache8_rows_weights_kernel"}),
    (BF, (8, 2, 128, 128, 64), [9, 1], True, {"cache8_attention_kernel", "cache8_rows_weights_kernel"}),
    (BF, (8, 2, 128, 128, 64), [130, 140], False, {"cache8_widen_kernel", "attention_prefill_kernel", "cache8_nan_kernel", "cache8_attention_kernel"}),
    (BF, (8, 2, 128, 128, 64), [130, 1], True, {"cache8_widen_kernel", "attention_prefill_kernel", "cache8_nan_kernel", "cache8_prompt_weights_kernel",
                                                "cache8_attention_kernel", "cache8_rows_weights_kernel"}),
])
def test_which_kernels_run(dtype, shape, lens, weights, want):
    from kernel_names import kernels
    from teenygrad_b200 import ops
    heads, kv, dim, vdim, block = shape
    cache, _ = filled(1, len(lens), kv, 300, dim, vdim, block, weights=weights)
    table, rows = rows_of(lens, range(len(lens)), [20] * len(lens))
    on, q = ops.step_table(table), rnd(2, rows, heads, dim).to(dtype).cuda()
    scratch, out = ops.cache8_attention_scratch(cache, on, q, weights), torch.zeros(rows, heads, vdim, dtype=dtype, device="cuda")
    got = kernels(lambda: ops.cache8_attention(q, cache, 0.1, on, weight_decay=0.5 if weights else None, out=out, scratch=scratch))
    assert all(any(w in name for name in got) for w in want) and all(any(w in name for w in want) for name in got), got


@DTYPES
def test_many_entries(dtype):
    """More entries than a warp counts at once, with empty ones in between, in slots far apart."""
    from teenygrad_b200 import ops
    n, slots, heads, kv, dim = 300, 70, 2, 1, 32
    cache, want = filled(3, slots, kv, 80, dim, dim, 16)
    table, row = [], 0
    for i in range(n):
        m = (1, 0, 2, 1, 1)[i % 5]
        table.append(((i * 37) % slots, (i * 11) % 78, row, m))
        row += m
    q = rnd(4, row, heads, dim).to(dtype)
    out = ops.cache8_attention(q.cuda(), cache, 0.2, ops.step_table(table))
    check(out, None, want.attention(q, 0.2, table), dtype, q, dim, 80, 0.0, table)


def test_prompts_of_more_entries_than_a_launch_takes():
    """130 prompts (128 to a launch), a few tokens between them, and slots so long that their widened tokens are held one at a time."""
    from teenygrad_b200 import ops
    heads, kv, dim = 6, 1, 16  # (prompts from 32 tokens on)
    cache, want = filled(5, 130, kv, 40, dim, dim, 16, weights=True)
    table, rows = rows_of([33 + i % 5 if i % 7 else 3 for i in range(130)], [(i * 3) % 130 for i in range(130)], [i % 3 for i in range(130)])
    q = rnd(6, rows, heads, dim).to(BF)
    out = ops.cache8_attention(q.cuda(), cache, 0.2, ops.step_table(table), weight_decay=0.0)
    ref = want.attention(q, 0.2, table, decay=0.0)
    check(out, None, ref, BF, q, dim, 40, 0.0, table)
    for slot, at, _, m in table:
        a, b = cache.weights[slot, 0, :at + m].double().cpu(), want.weights[slot, 0, :at + m]
        assert float(((a - b).abs() / (b + 1e-30)).max()) < 1e-4
    long, plain = filled(7, 3, 2, 40000, 32, 16, 128)
    table, rows = rows_of([70, 130, 65], [2, 0, 1], [300, 0, 39935])
    plain.k, plain.v = plain.k[:, :1], plain.v[:, :1]
    q = rnd(8, rows, 8, 32).to(BF)
    out = ops.cache8_attention(q.cuda(), long, 0.2, ops.step_table(table))
    ref = plain.attention(q[:, :4], 0.2, table)  # (the first kv head's query heads)
    check(out[:, :4], None, ref, BF, q[:, :4], 32, 40000, 0.0, table)


@DTYPES
@pytest.mark.parametrize("n", [1, 70])
def test_a_cache_of_more_than_four_billion_bytes(dtype, n):
    """The last slot of a cache whose offsets need more than 32 bits: append, attention, eviction."""
    from teenygrad_b200 import ops
    heads, kv, dim, slots, cap = 4, 2, 128, 3, 6_000_000
    cache = ops.cache8(slots, kv, cap, dim, 16, 128, weights=True)
    want = oc.Cache(torch.zeros(1, kv, n + 9, dim, dtype=torch.uint8), torch.zeros(1, kv, n + 9, 16, dtype=torch.uint8), torch.zeros(1, kv, 1), torch.zeros(1, kv, 1),
                    128, torch.zeros(1, kv, n + 9))
    q, k, v = (rnd(90 + i, n, h, d).to(dtype) for i, (h, d) in enumerate(((heads, dim), (kv, dim), (kv, 16))))
    far, near = ops.step_table([(2, 0, 0, n)]), [(0, 0, 0, n)]
    ops.cache8_append(cache, k.cuda(), v.cuda(), far)
    want.append(k, v, near)
    out = ops.cache8_attention(q.cuda(), cache, 0.1, far, weight_decay=0.0)
    check(out, None, want.attention(q, 0.1, near, decay=0.0), dtype, q, dim, n, 0.0, near)
    assert float((cache.weights[2, :, :n].double().cpu() - want.weights[0, :, :n]).abs().max()) < 1e-4
    want.weights[0, :, :n] = cache.weights[2, :, :n].double().cpu()
    kept = ops.cache8_evict(cache, ops.step_table([(2, n, 0, 0)]), max(1, n // 2), n // 8)
    assert torch.equal(kept.cpu(), want.evict([(0, n, 0, 0)], max(1, n // 2), n // 8))
    assert torch.equal(cache.k[2, :, :n].view(torch.uint8).cpu() & 127, want.k[0, :, :n] & 127)
    del cache
    torch.cuda.empty_cache()


@DTYPES
@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("lens", [[1, 1], [5, 150]])
def test_views_of_queries_outputs_and_gates(dtype, offset, lens):
    """Rows inside wider ones, and rows that do not start on 16 bytes."""
    from teenygrad_b200 import ops
    heads, kv, dim, vdim = 4, 2, 64, 48
    cache, want = filled(9, 2, kv, 200, dim, vdim, 32)
    table, rows = rows_of(lens, [1, 0], [40, 7])
    wide = rnd(10, rows, heads * (dim + 2 * vdim) + 8 + offset).to(dtype).cuda()
    q = wide[:, offset:offset + heads * dim].unflatten(1, (heads, dim))
    out = wide[:, offset + heads * dim:offset + heads * (dim + vdim)].unflatten(1, (heads, vdim))
    gate = wide[:, offset + heads * (dim + vdim):offset + heads * (dim + 2 * vdim)]
    qc, gc, rest = q.cpu().clone(), gate.cpu().clone(), wide[:, offset + heads * (dim + 2 * vdim):].clone()
    ops.cache8_attention(q, cache, 0.1, ops.step_table(table), gate=gate, out=out)
    check(out, None, want.attention(qc, 0.1, table, gate=gc), dtype, qc, dim, 200, 0.0, table)
    assert torch.equal(q.cpu(), qc) and torch.equal(gate.cpu(), gc) and torch.equal(rest, wide[:, offset + heads * (dim + 2 * vdim):])


@DTYPES
@pytest.mark.parametrize("lens", [[1, 3], [140, 2]])
def test_without_the_hosts_table(dtype, lens):
    """The C entry points with the table on the device alone: the same bits."""
    from teenygrad_b200 import ops
    from teenygrad_b200._lib import lib
    heads, kv, dim = 8, 2, 64
    cache, _ = filled(11, 2, kv, 200, dim, dim, 32)
    table, rows = rows_of(lens, [1, 0], [40, 7])
    on, q = ops.step_table(table), rnd(12, rows, heads, dim).to(dtype).cuda()
    scratch = ops.cache8_attention_scratch(cache, on, q)
    want, got = ops.cache8_attention(q, cache, 0.1, on, scratch=scratch), torch.zeros(rows, heads, dim, dtype=dtype, device="cuda")
    args = [int(dtype == F32), *cache._at, None, 0.0, q.data_ptr(), heads * dim, got.data_ptr(), heads * dim, rows, heads, 0.1, 0.0, None, None, 0, None,
            scratch.data_ptr(), scratch.numel(), on.seqs.data_ptr(), None, on.n, on.longest, ops._stream()]
    assert lib.teeny_cache8_attention(*args) == 0
    assert torch.equal(want, got)


@DTYPES
@pytest.mark.parametrize("lens", [[1, 3], [140, 2]])
def test_a_bound_that_nothing_reaches(dtype, lens):
    """max_len far above the longest entry, without the host's table."""
    from teenygrad_b200 import ops
    from teenygrad_b200._lib import lib
    heads, kv, dim, most = 8, 2, 64, 2 ** 31 - 1
    cache, want = filled(17, 2, kv, 200, dim, dim, 32)
    table, rows = rows_of(lens, [1, 0], [40, 7])
    on = ops.step_table(table)
    q, k, v = (rnd(18 + i, rows, h, dim).to(dtype) for i, h in enumerate((heads, kv, kv)))
    x, kx, vx, out = q.cuda(), k.cuda(), v.cuda(), torch.zeros(rows, heads, dim, dtype=dtype, device="cuda")
    f32, tail = int(dtype == F32), [on.seqs.data_ptr(), None, on.n, most, ops._stream()]
    assert lib.teeny_cache8_append(f32, *cache._at, None, kx.data_ptr(), kv * dim, vx.data_ptr(), kv * dim, rows, *tail) == 0
    want.append(k, v, table)
    same(cache, want)
    size = lib.teeny_cache8_attention_scratch_bytes(cache._shape_at, f32, heads, rows, on.n, most, 0)
    scratch = torch.zeros(size, dtype=torch.uint8, device="cuda")
    assert lib.teeny_cache8_attention(f32, *cache._at, None, 0.0, x.data_ptr(), heads * dim, out.data_ptr(), heads * dim, rows, heads, 0.1, 0.0, None, None, 0,
                                      None, scratch.data_ptr(), size, *tail) == 0
    check(out, None, want.attention(q, 0.1, table), dtype, q, dim, 200, 0.0, table)


@DTYPES
def test_calls_of_any_sizes_share_scratch(dtype):
    from teenygrad_b200 import ops
    cache, want = filled(17, 6, 2, 700, 64, 64, 16, weights=True)
    calls = []
    for lens, pos in (([1] * 6, [699, 0, 64, 300, 31, 500]), ([1], [650]), ([9, 1, 140, 2, 0, 3], [100, 5, 300, 690, 7, 400]), ([200], [3]), ([5, 5], [600, 2])):
        table, rows = rows_of(lens, range(len(lens)), pos)
        calls.append((table, ops.step_table(table), rnd(18 + rows, rows, 8, 64).to(dtype)))
    size = max((ops.cache8_attention_scratch(cache, on, q, True) for _, on, q in calls), key=lambda t: t.numel())
    scratch = torch.full((size.numel(),), 255, dtype=torch.uint8, device="cuda")
    scratch[:4096] = 0
    gone = ops.step_table([(5, 60, 0, 0)])
    for turn in range(3):
        for i in (0, 2, 1, 3, 0, 4, 2):
            table, on, q = calls[i]
            out = ops.cache8_attention(q.cuda(), cache, 0.1, on, weight_decay=0.0, scratch=scratch)
            if turn == 0:
                check(out, None, want.attention(q, 0.1, table), dtype, q, 64, 700, 0.0, table)
                calls[i] = (table, on, q)
            if i == 1:
                ops.cache8_evict(cache, gone, 60, 0, scratch=scratch)  # (all of them are kept)
                if turn == 0:
                    want.weights.copy_(cache.weights)
                    want.evict([(5, 60, 0, 0)], 60, 0)
    assert not bool(scratch[:4096].any())


@DTYPES
@pytest.mark.parametrize("lens", [[1, 1, 1], [4, 140, 1]])
def test_the_same_call_gives_the_same_bits(dtype, lens):
    from teenygrad_b200 import ops
    cache, _ = filled(13, 3, 2, 900, 128, 128, 64, weights=True)
    table, rows = rows_of(lens, [1, 0, 2], [700, 300, 5])
    on, q = ops.step_table(table), rnd(14, rows, 8, 128).to(dtype).cuda()
    scratch = ops.cache8_attention_scratch(cache, on, q, True)
    first = ops.cache8_attention(q, cache, 0.1, on, weight_decay=0.0, scratch=scratch)
    w = cache.weights.clone()
    for _ in range(20):
        assert torch.equal(ops.cache8_attention(q, cache, 0.1, on, weight_decay=0.0, scratch=scratch), first) and torch.equal(cache.weights, w)


def test_a_soft_cap_far_above_the_scores():
    """tanh near zero: the capped scores are the scores, up to f32's roundings."""
    from teenygrad_b200 import ops
    for lens in ([1, 1], [120, 1]):
        cache, want = filled(15, 2, 2, 200, 64, 64, 32, weights=True)
        table, rows = rows_of(lens, [1, 0], [60, 150])
        for dtype in (F32, BF):
            q = rnd(16, rows, 8, 64).to(dtype)
            ops.cache8_attention(q.cuda(), cache, 0.1, ops.step_table(table), softcap=3e4, weight_decay=0.0)
            ref = want.attention(q, 0.1, table, 3e4, decay=0.0)
            near = float(bounds(dtype, ref, q, 64, 200, 0.0)[2].max()) + (rows * 4 + 4) * 2.0 ** -24  # (no term for the cap)
            for slot, at, _, m in table:
                a, b = cache.weights[slot, :, :at + m].double().cpu(), want.weights[slot, :, :at + m]
                assert float(((a - b).abs() / b).max()) < near


@DTYPES
@pytest.mark.parametrize("lens", [[1, 1], [5, 1], [130, 1]])
@pytest.mark.parametrize("softcap", [2e-30, 1e-6])
def test_a_soft_cap_far_below_the_scores(dtype, lens, softcap):
    """Every score is the cap or its negative: nearly equal probabilities."""
    attend(dtype, (4, 2, 64, 64, 32), lens, [60, 150][:len(lens)], 200, softcap, decay=0.5, seed=19)


# ------------------------------------------------------------------------------------------------ evict
@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (50, 0), (50, 50), (130, 17), (299, 5), (300, 10)])
def test_evict(block, keep, recent):
    from teenygrad_b200 import ops
    cache, want = filled(keep, 5, 2, 300, 64, 48, block, weights=True)
    lens = [300, 131, 50, 1, 0]
    table = [(s, n, 0, 0) for s, n in zip([3, 0, 4, 1, 2], lens)]
    kept = ops.cache8_evict(cache, ops.step_table(table), keep, recent)
    assert torch.equal(kept.cpu(), want.evict(table, keep, recent))
    same(cache, want)


def test_evict_ties_and_weights_that_are_not_numbers():
    from teenygrad_b200 import ops
    cache, want = filled(3, 2, 4, 5000, 16, 16, 16, weights=True)
    w = torch.randint(0, 4, (2, 4, 5000), generator=torch.Generator().manual_seed(1)).float()
    w[:, 0] = 1.0
    w[:, 1, ::2], w[:, 1, 1::2] = 0.0, -0.0
    w[:, 2, 5:4000], w[:, 2, 7], w[:, 2, 9], w[:, 2, 4500] = float("nan"), -float("inf"), float("inf"), float("inf")
    w[0, 3] = 1e-40 * torch.arange(5000).flip(0)
    want.weights.copy_(w)
    cache.weights.copy_(w)
    table = [(1, 4999, 0, 0), (0, 5000, 0, 0)]
    kept = ops.cache8_evict(cache, ops.step_table(table), 1500, 100)
    assert torch.equal(kept.cpu(), want.evict(table, 1500, 100))
    same(cache, want)


@pytest.mark.parametrize("n,keep,recent", [(3000, 2999, 7), (17000, 40, 0), (40000, 20000, 64)])
def test_evict_long(n, keep, recent):
    """Candidates that a thread holds 16 of, and more than it holds at all; pieces that wait for many others."""
    from teenygrad_b200 import ops
    cache, want = filled(n, 2, 1, n, 32, 16, 128, weights=True)
    w = torch.exp(2 * rnd(1, 2, 1, n))
    w[:, :, 3:n // 2:2] = 0.25  # (many equal ones around the border)
    want.weights.copy_(w)
    cache.weights.copy_(w)
    table = [(1, n, 0, 0), (0, n - 1, 0, 0)]
    kept = ops.cache8_evict(cache, ops.step_table(table), keep, recent)
    assert torch.equal(kept.cpu(), want.evict(table, keep, recent))
    same(cache, want)


# ------------------------------------------------------------------------------------------------ together
@DTYPES
def test_a_sequence_that_is_thinned_out_while_it_grows(dtype):
    """Prompts into the cache, attention that counts weights, eviction down to a budget, single tokens behind it, another eviction: each step from
    the GPU's own cache, whose content is checked against the restatement at every step."""
    from teenygrad_b200 import ops
    heads, kv, dim, vdim, block, cap, budget = 4, 2, 64, 32, 32, 220, 90
    cache = ops.cache8(2, kv, cap, dim, vdim, block, weights=True)
    state = lambda: oc.Cache(cache.k.view(torch.uint8).cpu(), cache.v.view(torch.uint8).cpu(), cache.k_scale.cpu(), cache.v_scale.cpu(), block,  # noqa: E731
                             cache.weights.cpu())
    live = [0, 0]

    def step(lens, seed):
        table, rows = rows_of(lens, [1, 0], [live[1], live[0]])
        q, k, v = (rnd(seed + i, rows, h, d).to(dtype) for i, (h, d) in enumerate(((heads, dim), (kv, dim), (kv, vdim))))
        want = state()
        on = ops.step_table(table)
        ops.cache8_append(cache, k.cuda(), v.cuda(), on)
        want.append(k, v, table)
        same(cache, want)
        out = ops.cache8_attention(q.cuda(), cache, 0.2, on, weight_decay=0.9)
        ref = want.attention(q, 0.2, table, decay=0.9)
        check(out, None, ref, dtype, q, dim, cap, 0.0, table)
        assert float((cache.weights.double().cpu() - want.weights).abs().max()) < 1e-4
        for slot, p, _, n in table:
            live[slot] = p + n

    def evict():
        want = state()
        table = [(s, live[s], 0, 0) for s in (0, 1)]
        kept = ops.cache8_evict(cache, ops.step_table(table), budget, 16)
        assert torch.equal(kept.cpu(), want.evict(table, budget, 16))
        same(cache, want)
        for s in (0, 1):
            live[s] = min(live[s], budget)

    step([200, 75], 100)
    evict()
    for i in range(3):
        step([1, 1], 200 + 10 * i)
    step([4, 7], 300)
    evict()
    step([1, 1], 400)


@DTYPES
def test_a_captured_step_follows_its_table(dtype):
    """Append, attention with weights and eviction in one graph, replayed after the table on the device has moved on: the same as the calls."""
    from teenygrad_b200 import ops
    heads, kv, dim, block = 8, 2, 128, 64
    one, _ = filled(51, 3, kv, 400, dim, dim, block, weights=True)
    two, _ = filled(51, 3, kv, 400, dim, dim, block, weights=True)
    entries = [(2, 100, 0, 1), (0, 17, 1, 1)]
    q, k, v = (rnd(60 + i, 2, h, dim).to(dtype).cuda() for i, h in enumerate((heads, kv, kv)))
    on, gone = ops.step_table(entries), ops.step_table([(1, 300, 0, 0)])

    def run(cache, out, kept):
        ops.cache8_append(cache, k, v, on)
        ops.cache8_attention(q, cache, 0.1, on, weight_decay=0.5, out=out)
        ops.cache8_evict(cache, gone, 120, 8, kept=kept)
    out, kept = torch.zeros(2, heads, dim, dtype=dtype, device="cuda"), torch.zeros(1, kv, 120, dtype=torch.int32, device="cuda")
    run(two, out, kept)  # (loads the kernels)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(one, out, kept)
    two, _ = filled(51, 3, kv, 400, dim, dim, block, weights=True)
    for move in ((0, 0), (200, 5), (98, 300)):
        on.seqs[0, 1], on.seqs[1, 1] = 100 + move[0], 17 + move[1]
        graph.replay()
        got, gotk = out.clone(), kept.clone()
        run(two, out, kept)
        assert torch.equal(got, out) and torch.equal(gotk, kept)
        for a, b in ((one.k, two.k), (one.v, two.v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(one.k_scale, two.k_scale) and torch.equal(one.weights, two.weights)


@DTYPES
@pytest.mark.parametrize("lens", [[150, 140], [9, 9]])
def test_a_captured_call_follows_its_tables_lengths(dtype, lens):
    """Entries that were captured long and are short when the graph is replayed, and the other way round."""
    from teenygrad_b200 import ops
    heads, kv, dim = 8, 2, 128
    table, rows = rows_of(lens, [1, 0], [40, 7])
    on, q = ops.step_table(table), rnd(81, rows, heads, dim).to(dtype)
    cache, _ = filled(82, 2, kv, 200, dim, dim, 32, weights=True)
    x, out = q.cuda(), torch.zeros(rows, heads, dim, dtype=dtype, device="cuda")
    ops.cache8_attention(x, cache, 0.1, on, weight_decay=0.5, out=out)  # (loads the kernels)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache8_attention(x, cache, 0.1, on, weight_decay=0.5, out=out)
    for now in ([1, 1], [lens[0], 1], [2, lens[1]], lens, [0, 3]):
        fresh, want = filled(82, 2, kv, 200, dim, dim, 32, weights=True)
        cache.weights.copy_(fresh.weights)
        entries = [(s, p, row, n) for (s, p, row, _), n in zip(table, now)]
        on.seqs.copy_(torch.tensor(entries, dtype=torch.int32))
        out.fill_(5.0)
        graph.replay()
        ref = want.attention(q, 0.1, entries, decay=0.5)
        check(out, None, ref, dtype, q, dim, 200, 0.0, entries)
        _, _, p = bounds(dtype, ref, q, dim, 200, 0.0)
        near = float(p.max()) + (max(lens) * heads // kv + 4) * 2.0 ** -24
        assert float(((cache.weights.double().cpu() - want.weights).abs() - near * want.weights).max()) <= 0.0, now
        mine = torch.zeros(rows, dtype=torch.bool)
        for _, _, row, n in entries:
            mine[row:row + n] = True
        assert bool((out.cpu()[~mine] == 5.0).all())


@DTYPES
def test_two_streams_at_once(dtype):
    """Calls of two streams, each with its own cache and scratch, give what they give alone."""
    from teenygrad_b200 import ops
    caches = [filled(70 + i, 4, 2, 900, 128, 128, 64, weights=True)[0] for i in range(2)]
    q = [rnd(80 + i, 4, 8, 128).to(dtype).cuda() for i in range(2)]
    table = ops.step_table([(i, 899 - 100 * i, i, 1) for i in range(4)])
    want = [ops.cache8_attention(q[i], caches[i], 0.1, table) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.cache8_attention(q[i], caches[i], 0.1, table))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
