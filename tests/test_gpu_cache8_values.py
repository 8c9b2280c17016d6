"""Attention over the 8-bit cache where its scales, queries and sinks are far from ordinary, and with bounds that follow each kernel's own roundings,
against the 64-bit restatement in oracle/cache8.py."""
import pytest
import torch

from test_gpu_cache8 import filled, rnd, rows_of, same

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DTYPES = pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    from teenygrad_b200 import ops
    assert ops.device_error() == 0


def visible_top(want, table, rows, heads):
    """Largest value scale that a row of a query head sees, [rows, heads]."""
    top, H = torch.zeros(rows, heads, dtype=torch.float64), want.k.shape[1]
    for slot, pos, row, n in table:
        for i in range(n):
            seen = want.vs[slot, :, :(pos + i) // want.block + 1].max(-1)[0]
            top[row + i] = seen.repeat_interleave(heads // H)
    return top


def limits(dtype, ref, table, dim, top, softcap=0.0, prompts=False):
    """How far right outputs, lse and (relatively) probabilities may be.

    A score is a sum of `dim` products in f32, cut off rather than rounded (2^-23 of the sum of magnitudes each); a bf16 query is one f16 term, exact down to 2^-28 of
    its row's largest number and off by 2^-39 of that below, an f32 one two terms (2^-22); five more f32 roundings of the score, its factor and its difference
    from the maximum; a soft cap 2^-20 of the cap.  A probability is off relatively by twice that (its own and the sum's) and by its exponential and the sums
    (2^-21 and 2^-24 a key).  Before the values' product it is rounded to f16 (2^-11; f32: two terms, 2^-22), in prompts' kernel to bf16 (2^-8), and f16 is
    off by 2^-25 at least, of 2^14 (two terms: 2^-50 altogether), in units of the largest scale the row sees, or 2^-112, times codes up to 448.  The output is rounded
    once (2^-8, 2^-24).  The factor behind the sums may be subnormal: off by 2^-150, for sums up to 2^23 a key."""
    out, lse, mass, dots = ref
    keys = max(p + n for _, p, _, n in table)
    score = torch.where(torch.isinf(lse), 0.0, lse).abs() + dots
    delta = dim * 2.0 ** -23 * dots + (2.0 ** -39 * dim if dtype == BF else 2.0 ** -22) * dots + 5 * 2.0 ** -24 * score + 2.0 ** -20 * softcap
    p = 2 * delta + 2.0 ** -21 + keys * 2.0 ** -24
    half, two = (2.0 ** -8, 2.0 ** -8 if prompts else 2.0 ** -11) if dtype == BF else (2.0 ** -24, 2.0 ** -22)
    least = keys * 448 * (2.0 ** -39 if dtype == BF else 2.0 ** -50) * top.clamp(min=2.0 ** -112)
    near = half * out.abs() + (two + p[..., None]) * 1.02 * mass + least[..., None] + keys * 2.0 ** -126
    return near, delta + p + 4 * 2.0 ** -24 * score, p


def run(dtype, cache, want, table, rows, heads, seed, factor=1.0, scale=None, sink=None, softcap=0.0, off16=False, decay=0.5):
    """One call with everything checked: rows of the table, lse, weights, the cache as it was."""
    from teenygrad_b200 import ops
    dim, vdim, kv = want.k.shape[3], want.v.shape[3], want.k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    q = (factor * rnd(seed, rows, heads, dim)).to(dtype)
    if off16:  # rows that do not start on 16 bytes: not the prompts' kernel
        wide = torch.zeros(rows, heads * dim + 1, dtype=dtype, device="cuda")
        x = wide[:, 1:].unflatten(1, (heads, dim))
        x.copy_(q)
    else:
        x = q.cuda()
    lse = torch.full((rows, heads), 3.0, device="cuda")
    out = ops.cache8_attention(x, cache, scale, ops.step_table(table), softcap=softcap, sink=None if sink is None else sink.cuda(),
                               weight_decay=decay, lse=lse)
    was = want.weights.clone()
    ref = want.attention(q, scale, table, softcap, sink, None, decay)
    longest = max(n for _, _, _, n in table)
    prompts = dtype == BF and not off16 and longest >= max(32, 192 // (heads // kv))
    near, nearz, p = limits(dtype, ref, table, dim, visible_top(want, table, rows, heads), softcap, prompts)
    got, z = out.double().cpu(), lse.double().cpu()
    for slot, pos, row, n in table:
        at = slice(row, row + n)
        assert bool(torch.isfinite(got[at]).all())
        assert float(((got[at] - ref[0][at]).abs() / near[at]).max()) <= 1.0
        inf = torch.isinf(ref[1][at])
        assert torch.equal(torch.isinf(z[at]), inf) and bool((z[at][inf] == ref[1][at][inf]).all())
        assert float(((z[at] - ref[1][at]).abs() / nearz[at])[~inf].max() if bool((~inf).any()) else 0.0) <= 1.0
        gw, ww = cache.weights[slot].double().cpu(), want.weights[slot]
        assert torch.equal(gw[:, pos + n:], was[slot, :, pos + n:])
        far = (gw - ww).abs()[:, :pos + n]
        finite, least = p[at][~inf], n * heads // kv * 2.0 ** -126  # (a subnormal probability counts as none)
        assert bool((far <= (float(finite.max() if finite.numel() else 0.0) + (n * heads // kv + 4) * 2.0 ** -24) * ww[:, :pos + n] + least).all())
    same(cache, want, weights=False)
    return got, z


def put(cache, want, name, slot, head, tokens, codes=None, scale=None):
    """Codes and block scales of a head's tokens, in both caches; whole blocks where a scale is given."""
    held, scales = getattr(want, name), getattr(want, name + "s")
    if codes is not None:
        held[slot, head, tokens] = codes
        getattr(cache, name).view(torch.uint8).copy_(held)
    if scale is not None:
        scales[slot, head, tokens.start // want.block:-(-tokens.stop // want.block)] = scale
        getattr(cache, name + "_scale").copy_(scales)


LENS = [([1, 1, 1], [0, 31, 149]), ([3, 1, 5], [0, 60, 140]), ([140, 40, 1], [0, 33, 90])]


@DTYPES
@pytest.mark.parametrize("lens,pos", LENS)
@pytest.mark.parametrize("zeros", ["first", "slice", "later", "head", "all"])
@pytest.mark.parametrize("heads,kv,dim,block,off16", [(8, 2, 64, 32, False), (4, 2, 128, 16, True), (32, 2, 64, 64, True)])
def test_values_of_zeros(dtype, lens, pos, zeros, heads, kv, dim, block, off16):
    """Tokens whose values are zeros, appended as such: their blocks have the least scale there is, and attention gives zeros for them and no NaN."""
    from teenygrad_b200 import ops
    cap, slots = 190, [1, 2, 0]
    cache, want = filled(60, 3, kv, cap, dim, 48, block, weights=True)
    every, rows = rows_of([p + n for p, n in zip(pos, lens)], slots, [0] * 3)
    k, v = rnd(61, rows, kv, dim), rnd(62, rows, kv, 48)
    for _, _, row, n in every:
        if zeros == "first":
            v[row] = 0.0
        elif zeros == "slice":
            v[row:row + min(n, 64)] = 0.0
        elif zeros == "later":
            v[row + min(n - 1, 64):row + n] = 0.0
        elif zeros == "head":
            v[row:row + n, 1] = 0.0
        else:
            v[row:row + n] = 0.0
    k, v = k.to(dtype), v.to(dtype)
    ops.cache8_append(cache, k.cuda(), v.cuda(), ops.step_table(every))
    want.append(k, v, every)
    same(cache, want)
    table, rows = rows_of(lens, slots, pos)
    got, _ = run(dtype, cache, want, table, rows, heads, 63, off16=off16)
    if zeros in ("head", "all"):
        for _, _, row, n in table:
            assert bool((got[row:row + n, heads // 2 if zeros == "head" else 0:] == 0.0).all())


@DTYPES
@pytest.mark.parametrize("lens,pos", LENS)
@pytest.mark.parametrize("exponents", [(-126,), (-115,), (-113, -112, -111), (-126, -9), (-9, -126), (100,), (-9, 5, -20, 11)])
def test_values_of_small_and_large_scales(dtype, lens, pos, exponents):
    """Scales from the least one on, the same for a sequence or from block to block."""
    heads, kv, dim, block, cap = 8, 2, 64, 32, 190
    cache, want = filled(64, 3, kv, cap, dim, 48, block, weights=True)
    for s in range(3):
        for h in range(kv):
            for b in range(-(-cap // block)):
                put(cache, want, "v", s, h, slice(b * block, min(cap, (b + 1) * block)), scale=2.0 ** exponents[(b + h) % len(exponents)])
    table, rows = rows_of(lens, [1, 2, 0], pos)
    run(dtype, cache, want, table, rows, heads, 65, off16=True)
    if min(exponents) > -100:  # (bf16 numbers below 2^-126 are subnormal where prompts hold them)
        run(dtype, cache, want, table, rows, heads, 66)


@DTYPES
@pytest.mark.parametrize("lens,pos", [([20, 9], [8, 41]), ([40, 3], [0, 14]), ([140, 150], [5, 0])])
@pytest.mark.parametrize("up", [40, 100])
@pytest.mark.parametrize("off16", [False, True])
def test_values_that_a_row_does_not_see_are_of_no_scale_to_it(dtype, lens, pos, up, off16):
    """The entry's later blocks are 2^up larger than what its first rows see."""
    heads, kv, dim, block, cap = 8, 2, 64, 16, 190
    cache, want = filled(67, 2, kv, cap, dim, 48, block, weights=True)
    table, rows = rows_of(lens, [1, 0], pos)
    for slot, p, _, n in table:
        at = min(-(-(p + 2) // block) * block, cap // block * block)  # the first block that the entry's first row does not see
        for h in range(kv):
            for b in range(at // block, -(-cap // block)):
                put(cache, want, "v", slot, h, slice(b * block, min(cap, (b + 1) * block)), scale=2.0 ** (up - 9 + (b & 1)))
    run(dtype, cache, want, table, rows, heads, 68, off16=off16)


@DTYPES
@pytest.mark.parametrize("lens,pos", LENS)
@pytest.mark.parametrize("sink", [60.0, 95.0, 150.0, 3e4, -150.0, float("inf"), -float("inf")])
def test_sinks_far_from_the_scores(dtype, lens, pos, sink):
    """lse is the sink's value where that is far above the scores, and theirs where it is far below."""
    heads, kv, dim = 8, 2, 64
    cache, want = filled(69, 3, kv, 190, dim, 48, 32, weights=True)
    table, rows = rows_of(lens, [1, 2, 0], pos)
    sinks = rnd(70, heads)
    sinks[1], sinks[3], sinks[6] = sink, sink, sink + 1.0
    run(dtype, cache, want, table, rows, heads, 71, sink=sinks)


@DTYPES
@pytest.mark.parametrize("lens,pos", LENS)
@pytest.mark.parametrize("q_exp,k_exp", [(117, -118), (124, -118), (-110, 100), (-100, 80)])
def test_queries_of_any_size(dtype, lens, pos, q_exp, k_exp):
    """Rows of queries near both ends of their type, over keys that make ordinary scores of them."""
    heads, kv, dim, cap = 8, 2, 64, 190
    cache, want = filled(72, 3, kv, cap, dim, 48, 32, weights=True)
    for s in range(3):
        for h in range(kv):
            put(cache, want, "k", s, h, slice(0, cap), scale=2.0 ** k_exp)
    table, rows = rows_of(lens, [1, 2, 0], pos)
    # (score_scale takes what is left: dots of about 2^(3 + 6.5 + q_exp + k_exp))
    run(dtype, cache, want, table, rows, heads, 73, factor=2.0 ** q_exp, scale=2.0 ** min(-9 - q_exp - k_exp, 20))


@DTYPES
@pytest.mark.parametrize("lens,pos", LENS)
@pytest.mark.parametrize("heads,kv,dim,block,off16", [(8, 2, 128, 64, False), (4, 4, 80, 16, True), (24, 2, 16, 32, True)])
def test_bounds_of_the_kernels_own_roundings(dtype, lens, pos, heads, kv, dim, block, off16):
    """Ordinary numbers: probabilities in f16 (prompts: bf16) or two terms of it, and nothing coarser."""
    cache, want = filled(74, 3, kv, 190, dim, 48, block, weights=True)
    table, rows = rows_of(lens, [1, 2, 0], pos)
    run(dtype, cache, want, table, rows, heads, 75, off16=off16, sink=rnd(76, heads), softcap=0.0 if off16 else 20.0)
