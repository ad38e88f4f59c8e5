"""Edges of the paged-cache operators on the GPU: what stands beside a row in memory,
weights at the ends of their range, and calls that share memory.  Tolerances are those of
test_paged_gpu.py, or equality of bits."""
import math

import pytest

from test_paged_gpu import (D, Setup, attention64, check_attention, check_verify, device_error, dtype_of, gen,  # noqa: F401
                            no_device_error, run_verify)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(cuda):
    import torch as _t
    return _t


@pytest.fixture(scope="module")
def P(cuda):
    from dial_cuda import paged
    return paged


# ------------------------------------------------------------------ verification
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [7, 777, 4099])
@pytest.mark.parametrize("bad", [math.nan, -0.05, -1e30, math.inf, -math.inf])
def test_draft_probs_of_rows_that_judge_no_draft_are_not_read(torch, P, dtype, V, bad):
    """A row of odd length shares its first and last vectors with its neighbours: the draft's
    weights in a sequence's last row and behind the last sequence may hold anything."""
    rows = [1, 2, 4, 0, 2, 3, 1, 2, 2, 5]
    g = gen(torch, V)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    R = start[-1] + 2
    logits = (torch.randn((R, V), generator=g, device="cuda") * 2).to(dtype_of(torch, dtype))
    draft = (logits.float() + torch.randn((R, V), generator=g, device="cuda")).softmax(-1)
    idle = [e - 1 for e, n in zip(start[1:], rows) if n] + [R - 2, R - 1]
    draft[idle] = 0
    ids = torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand((len(rows),), generator=g, device="cuda")
    accept = torch.full((R,), 0.999, device="cuda")
    want = check_verify(torch, P, logits, ids, start, [1.0] * len(rows), accept, u, draft)
    draft[idle] = bad
    got = run_verify(torch, P, logits, ids, start, [1.0] * len(rows), accept, u, draft)
    n = start[-1]
    assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1], want[1]) and torch.equal(got[2][:n], want[2][:n])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("step", [1, 7, 13])
@pytest.mark.parametrize("V", [1000, 151936])
def test_weights_that_count_only_together_draw_one_of_their_own(torch, P, dtype, rows, step, V):
    """Eight weights of e^-617.3, each below 2^-890 of the maximum's and above it as a sum, in one
    vector or several: with u = 0 one of them or the maximum is drawn, none without probability."""
    logits = torch.full((rows, V), -math.inf, device="cuda")
    at = 16 + step * torch.arange(8, device="cuda")
    logits[:, at] = -1
    logits[:, 900] = 0
    got = run_verify(torch, P, logits.to(dtype_of(torch, dtype)), [2] * rows, [0, rows], [1 / 617.3], [0.5] * rows, [0.0])
    assert int(got[0][0]) in at.tolist() + [900]
    assert got[1].tolist() == [1] and math.isfinite(float(got[2][0]))


@pytest.mark.parametrize("T", [1.0, 0.6])
@pytest.mark.parametrize("V", [1024, 9001])
def test_a_draft_nearly_equal_to_the_target(torch, P, T, V):
    """All of max(p - q, 0) but 2^-11.5 of it lies in weights of 2^-22.5 p, on which a sum of e in
    f32 cannot decide: at u = 0 and little above the first of them are drawn, as defined."""
    n = 64
    g = gen(torch, V)
    logits = torch.randn((2 * n, V), generator=g, device="cuda") * 2
    logits[:, V - 1] = logits[:, :V - 2].amax(-1) + 1
    p = (logits.double() / T).softmax(-1)
    draft = p * (1 - 2.0 ** -22.5)
    draft[:, V - 1] = p[:, V - 1] - 2.0 ** -11.5
    draft[:, V - 2] = p[:, V - 2] + 2.0 ** -11.5
    ids = torch.full((2 * n,), V - 2, dtype=torch.int32, device="cuda")
    u = torch.cat([torch.zeros(n // 2, device="cuda"), torch.rand(n // 2, generator=g, device="cuda") * 2.0 ** -11])
    temp = torch.full((n,), T, device="cuda")
    p = (logits.double() / temp[0].double()).softmax(-1)
    keep = (p[:, V - 2] < 0.9999 * draft[:, V - 2]).all()
    assert keep  # the draft is refused
    check_verify(torch, P, logits, ids, list(range(0, 2 * n + 1, 2)), temp, torch.full((2 * n,), 0.9999, device="cuda"), u,
                 draft.float())


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("octaves", [18, 22, 24])
@pytest.mark.parametrize("q,kv", [([1], [2049]), ([1, 2], [40001, 700]), ([5], [9000]), ([40], [2100]), ([300, 9], [2500, 5000])])
@pytest.mark.parametrize("dtype,quant", [("f16", False), ("bf16", False), ("f16", True), ("bf16", True)])
def test_a_first_key_that_takes_nearly_all_weight(torch, P, octaves, q, kv, dtype, quant):
    """The first key `octaves` above all others, with a value row of zeros (int8: a small one, as zeros
    have the scale 1): what the others leave is as exact as anywhere."""
    s = Setup(torch, P, q, kv, dtype, quant, 64, 2, seed=octaves)
    x = torch.randn((s.T, 8, D), generator=gen(torch, 5), device="cuda") * 0.3
    x[..., 0] = 4
    x = x.to(dtype_of(torch, dtype))
    at = octaves / (4 * D ** -0.5 * math.log2(math.e))
    s.pages[0][..., 0] = 0
    for b in range(len(q)):
        first = s.host_table[b][0]
        s.pages[0][first, :, 0] = 0
        s.pages[0][first, :, 0, 0] = 127 if quant else at
        if quant:
            s.scales[0][first, :, 0], s.scales[1][first, :, 0] = at / 127, 2.0 ** -12
        else:
            s.pages[1][first, :, 0] = 0
    check_attention(torch, s, x, s.cache.attention(x, s.batch))


@pytest.mark.parametrize("top", [2.0 ** 100, 2.0 ** 112, 2.0 ** 119, -2.0 ** 100, -2.0 ** 112, -2.0 ** 119, 2.0 ** -100, -2.0 ** -100])
@pytest.mark.parametrize("q,kv", [([1], [50]), ([3], [2100]), ([30, 1], [99, 700])])
def test_bf16_queries_at_the_ends_of_their_range_over_int8_pages(torch, P, top, q, kv):
    """One large value a query, every score of one sign: the key with the largest takes all."""
    s = Setup(torch, P, q, kv, "bf16", True, 32, 2)
    x = torch.zeros((s.T, 8, D), device="cuda")
    x[..., 3] = top
    x = x.bfloat16()
    s.pages[0].abs_().clamp_(min=1)
    check_attention(torch, s, x, s.cache.attention(x, s.batch))


@pytest.mark.parametrize("dtype,top,size", [("f16", 65504, 2e4), ("f16", -65504, 2e4), ("f16", -65504, 300), ("f16", 6e3, 2e4)] +
                         [("bf16", x * 2.0 ** e, 1) for x in (1, -1) for e in (24, 30, 100, 112, 119)])
@pytest.mark.parametrize("q,kv", [([1], [50]), ([3, 1], [2100, 77]), ([30, 1], [99, 700]), ([300], [3000])])
def test_scores_whose_last_bit_is_above_one(torch, P, dtype, top, size, q, kv):
    """Scores of 2^24 and more, exact in f32 and all of one sign: their factor rounds by octaves,
    and the key with the largest takes all."""
    s = Setup(torch, P, q, kv, dtype, False, 32, 2)
    x = torch.zeros((s.T, 8, D), device="cuda")
    x[..., 3] = top
    s.pages[0][..., 3] = (torch.rand(s.pages[0].shape[:3], generator=gen(torch, 6), device="cuda") * size + size / 8).to(s.pages[0].dtype)
    x = x.to(s.pages[0].dtype)
    check_attention(torch, s, x, s.cache.attention(x, s.batch))


@pytest.mark.parametrize("q,kv", [([6], [300]), ([70, 40], [300, 141]), ([1], [4000])])
@pytest.mark.parametrize("dtype,quant,bad,whole", [("bf16", False, b, w) for b in (math.nan, math.inf, -math.inf) for w in (True, False)] +
                         [("f16", False, b, False) for b in (math.nan, math.inf, -math.inf)] +
                         [("bf16", True, math.nan, True), ("f16", True, math.nan, True)])
@pytest.mark.parametrize("back", [1, 2, 3, 6, 150])
def test_a_key_that_is_not_finite(torch, P, q, kv, dtype, quant, bad, whole, back):
    """One key row, or one value of it, of kv head 0: tokens that see it have what the definition
    gives them, NaN or what the other keys give, the others nothing of it."""
    s = Setup(torch, P, q, kv, dtype, quant, 64, 2)
    at = kv[0] - back
    page, row = s.host_table[0][at // 64], at % 64
    if quant:
        s.scales[0][page, 0, row] = bad
    else:
        s.pages[0][page, 0, row, slice(None) if whole else 9] = bad
    x = torch.randn((s.T, 8, D), generator=gen(torch, 4), device="cuda").to(dtype_of(torch, dtype))
    got = s.cache.attention(x, s.batch)
    want, size = attention64(torch, s, x, D ** -0.5)
    nan = torch.isnan(want)
    sees = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
    sees[max(0, q[0] - back):q[0], :4] = True
    assert not nan[~sees].any() and (nan[sees].all() if whole else True)
    assert torch.equal(torch.isnan(got), nan)
    u = torch.finfo(x.dtype).eps / 2
    off = (got.double() - want).abs()
    assert torch.all((off <= u * want.abs() + (u + 2.0 ** -12) * size + 1e-7) | nan)
