"""The operators on paged latents, beams and cache moves against float64 restatements (tests/paged_ref.py).

Tolerances count roundings.  One rounding of a value to bf16 is off by at most 2^-8 of it, to fp32 by 2^-24; a sum of n
products in fp32 by n 2^-24 of the sum of their magnitudes.
"""

from __future__ import annotations

import random

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
E32 = 2.0 ** -24
SCALE = 128 ** -0.5


def _dev(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _within(got, want, tol):
    assert got.shape == want.shape
    assert torch.isfinite(got.float()).all()
    err = (got.double().cpu() - want).abs()
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((err / tol).max()):.2f} x the tolerance"


# ------------------------------------------------------------------ attention
def _attn_tol(want, mass, size, dtype, rank, keys):
    # scores: `rank` products (and the scale) in fp32, two of them in each probability (with the maximum); exponentials to
    # 2^-22; the sums over keys in fp32, of up to 2 keys values each (two parts of a probability)
    p = (2 * (rank + 4) * E32 * size + 2.0 ** -21)[..., None] * 2 * mass + (2 * keys + 700) * E32 * mass
    if dtype == F32:
        return p + E32 * want.abs() + 1e-30
    # a probability as two bf16 numbers: 2^-8 of 2^-8 of it is lost; and the result's rounding
    return p + 2.0 ** -16 * mass + 2.0 ** -8 * want.abs() + 1e-30


def _attn(c, *, slots="own", max_new=None, max_len=None, splits=0, out=None, scale=SCALE):
    from sophia_amd import ops
    slots = c.slots if isinstance(slots, str) else slots
    max_new = max(c.news) if max_new is None else max_new
    dt = c.qa.dtype
    if out is None:
        out = torch.full(c.qa.shape, 7.0, dtype=dt, device="cuda")
    qa, pages, table, cu, kv, sl = _dev(c.qa, c.pages, c.table, c.cu, c.kv_len, slots)
    got = ops.mla_paged_attn(qa, pages, table, cu, kv, scale, max_new=max_new, max_len=max_len, slots=sl, splits=splits, out=out)
    assert got is out
    want, mass, size, written = ref.attn(c.qa, c.pages, c.table, c.cu, c.kv_len, slots, scale, max_new)
    tol = _attn_tol(want, mass, size, dt, c.qa.size(2), max(c.lens + [1]))
    _within(got[written.cuda()], want[written], tol[written])
    assert (got[~written.cuda()] == 7.0).all(), "rows of no sequence were written"
    return got


ATTN = [
    dict(news=[1], lens=[1]),
    dict(news=[1], lens=[2]),
    dict(news=[1, 1, 1], lens=[63, 64, 65]),
    dict(news=[1] * 7, lens=[31, 32, 33, 127, 128, 129, 700]),
    dict(news=[1, 1], lens=[4100, 1500], page=64),
    dict(news=[2, 1, 2], lens=[2, 300, 301]),
    dict(news=[3], lens=[3]),
    dict(news=[7, 9], lens=[63, 200]),
    dict(news=[64], lens=[64], page=64),
    dict(news=[129], lens=[129], page=128),
    dict(news=[40, 1, 0, 17], lens=[300, 65, 12, 17]),
    dict(news=[33, 1, 8], lens=[1200, 1, 77], page=32),
    dict(news=[5, 1], lens=[70, 3], page=1),
    dict(news=[5, 1], lens=[70, 30], page=4),
    dict(news=[6, 1], lens=[900, 1000], page=1024),
    dict(news=[1, 1], lens=[300, 77], heads=1),
    dict(news=[40, 200], lens=[100, 200], heads=1),
    dict(news=[9, 1, 2], lens=[9, 140, 90], heads=5),
    dict(news=[1, 2], lens=[100, 333], heads=33),
    dict(news=[1, 3], lens=[70, 65], heads=128),
    dict(news=[1, 4, 70], lens=[200, 65, 130], rank=32),
    dict(news=[1, 4, 20], lens=[200, 65, 130], rank=64, heads=8),
    dict(news=[1, 4, 20], lens=[200, 65, 130], rank=256, heads=12),
    dict(news=[1] * 70, lens=[(37 * i) % 200 + 1 for i in range(70)], heads=2),
    dict(news=[(5 * i) % 7 for i in range(130)], lens=[(37 * i) % 90 + 7 for i in range(130)], heads=8, rank=32),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(f"{k}{str(v)[:24]}" for k, v in c.items()))
def test_attention_matches_float64(case, dtype):
    _attn(ref.Paged(**case, dtype=dtype, behind=3))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("splits", [1, 2, 3, 9, 64])
def test_attention_is_the_same_however_its_keys_are_divided(splits, dtype):
    _attn(ref.Paged([1, 30, 1, 2], [900, 700, 3, 513], dtype=dtype, page=32), splits=splits)


def test_a_bound_below_the_lengths_changes_nothing():
    for splits in (0, 1, 4):
        _attn(ref.Paged([1, 30, 1], [900, 700, 3], page=32), max_len=100, splits=splits)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_attention_without_keys_and_past_the_table(dtype):
    """Lengths of 0, shorter than the new tokens, negative, and past what the table holds; slots out of range."""
    c = ref.Paged([1, 5, 5, 1, 20, 1], [0, 3, 5, 40, 40, 64], dtype=dtype, spare=0)
    c.kv_len[0], c.kv_len[1] = -4, 3
    c.kv_len[3], c.kv_len[4] = 900, 2 ** 40
    c.slots[5] = 99
    c.pages = torch.where(torch.isnan(c.pages), 0.25, c.pages).to(dtype)     # (lengths past a sequence's own see what lies there)
    c.lens[3], c.lens[4] = 64, 64
    _attn(c)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_pages_that_are_none_hide_their_keys(dtype):
    """Holes as a sliding window leaves them, ids past the pool, a sequence with holes alone."""
    c = ref.Paged([1, 33, 1, 4], [500, 300, 90, 70], dtype=dtype)
    c.table[int(c.slots[0]), :20] = -1
    c.table[int(c.slots[1]), 3:9] = 10 ** 6
    c.table[int(c.slots[1]), 12] = -(2 ** 31)
    c.table[int(c.slots[2]), :] = -1
    _attn(c)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,news", [(16, [40]), (5, [6]), (16, [2]), (1, [100])])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_latent_that_is_not_finite_reaches_no_row_before_it(heads, news, value, dtype):
    c = ref.Paged(news, [news[0] + 70], heads=heads, dtype=dtype)
    at = c.lens[0] - (news[0] + 1) // 2            # in the middle of the new tokens
    page, row = c.place(0, at)
    clean = c.pages.clone()
    c.pages[page, row, 5] = value
    from sophia_amd import ops
    args = _dev(c.qa, c.pages, c.table, c.cu, c.kv_len)
    got = ops.mla_paged_attn(*args, SCALE, max_new=news[0], slots=c.slots.cuda()).cpu()
    before = at - (c.lens[0] - news[0])
    want, mass, size, _ = ref.attn(c.qa, clean, c.table, c.cu, c.kv_len, c.slots, SCALE, news[0])
    tol = _attn_tol(want, mass, size, dtype, 128, c.lens[0])
    _within(got[:before], want[:before], tol[:before])
    assert (~torch.isfinite(got[before:].float())).any(-1).all()


def test_rows_past_max_new_are_left_and_offsets_may_leave_rows_out():
    c = ref.Paged([9, 1, 4], [40, 20, 4])
    _attn(c, max_new=3)
    c.cu = torch.tensor([2, 7, 8, 12], dtype=torch.int32)      # rows 0, 1, 12, 13 belong to nobody
    c.news = [5, 1, 4]
    _attn(c)


def test_offsets_past_the_rows_stay_within_them():
    """Descending and too large offsets: nothing outside the tensors is touched."""
    from sophia_amd import ops
    c = ref.Paged([4, 4], [40, 20])
    qa, pages, table, kv, sl = _dev(c.qa, c.pages, c.table, c.kv_len, c.slots)
    for cu in ([0, 4, 2 ** 30], [-5, 4, 8], [8, 4, 0], [2 ** 30, 2 ** 30, 2 ** 30]):
        room = torch.full((24, 16, 128), 7.0, dtype=BF, device="cuda")
        ops.mla_paged_attn(qa, pages, table, torch.tensor(cu, dtype=torch.int32).cuda(), kv, SCALE, max_new=8, slots=sl, out=room[8:16])
        torch.cuda.synchronize()
        assert (room[:8] == 7.0).all() and (room[16:] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_strided_queries_outputs_and_pages(dtype):
    c = ref.Paged([1, 12], [50, 90], dtype=dtype)
    rows = c.rows
    wide = torch.zeros(rows, 17 * 128 + 8, dtype=dtype)
    wide[:, 8:8 + 16 * 128] = c.qa.view(rows, -1)
    c.qa = wide[:, 8:8 + 16 * 128].view(rows, 16, 128)
    two = torch.zeros(c.pages.size(0), 2, 16, 128, dtype=dtype)         # another layer's pages beside these
    two[:, 1] = c.pages
    c.pages = two[:, 1]
    from sophia_amd import ops
    dw, dp = wide.cuda(), two.cuda()
    out = torch.full((rows, 3, 16, 128), 7.0, dtype=dtype, device="cuda")
    got = ops.mla_paged_attn(dw[:, 8:8 + 16 * 128].view(rows, 16, 128), dp[:, 1], *_dev(c.table, c.cu, c.kv_len), SCALE, max_new=12,
                             slots=c.slots.cuda(), out=out[:, 1])
    want, mass, size, _ = ref.attn(c.qa, c.pages, c.table, c.cu, c.kv_len, c.slots, SCALE, 12)
    _within(got, want, _attn_tol(want, mass, size, dtype, 128, 90))
    assert (out[:, 0] == 7.0).all() and (out[:, 2] == 7.0).all()


def test_sequences_share_pages_and_large_scores_stay_exact():
    c = ref.Paged([1, 1, 3], [200, 200, 203], q_std=40.0)
    c.table[int(c.slots[1])] = c.table[int(c.slots[0])]
    c.table[int(c.slots[2]), :12] = c.table[int(c.slots[0]), :12]
    _attn(c)


def test_a_pool_past_32_bit_offsets():
    """Pages of a pool of more than 2^31 values (4.3 GB)."""
    from sophia_amd import ops
    n = 2 ** 31 // (64 * 128) + 40
    pool = torch.zeros(n, 64, 128, dtype=BF, device="cuda")
    c = ref.Paged([1, 10], [100, 90], page=64)
    ids = torch.unique(c.table[c.table >= 0]).tolist()
    far = {p: n - 1 - i for i, p in enumerate(ids)}
    for p in ids:
        pool[far[p]] = c.pages[p].cuda()
    table = torch.tensor([[far.get(int(v), -1) for v in row] for row in c.table], dtype=torch.int32)
    got = ops.mla_paged_attn(c.qa.cuda(), pool, *_dev(table, c.cu, c.kv_len), SCALE, max_new=10, slots=c.slots.cuda())
    want, mass, size, _ = ref.attn(c.qa, c.pages, c.table, c.cu, c.kv_len, c.slots, SCALE, 10)
    _within(got, want, _attn_tol(want, mass, size, BF, 128, 100))


def test_attention_of_nothing():
    from sophia_amd import ops
    c = ref.Paged([1], [5])
    pages, table = _dev(c.pages, c.table)
    i32, i64 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.int64, device="cuda")
    for rows, cu in ((0, [0, 0]), (3, [0])):
        out = torch.full((rows, 16, 128), 7.0, dtype=BF, device="cuda")
        qa = torch.zeros(rows, 16, 128, dtype=BF, device="cuda")
        ops.mla_paged_attn(qa, pages, table, torch.tensor(cu, **i32), torch.zeros(len(cu) - 1, **i64), SCALE, max_new=1, out=out)
        assert (out == 7.0).all()


# ------------------------------------------------------------------ norms
NORMS = [dict(news=[1], lens=[1]), dict(news=[1] * 70, lens=[3 * i + 1 for i in range(70)]), dict(news=[40, 0, 3, 17], lens=[90, 5, 3, 64]),
         dict(news=[5, 2], lens=[70, 30], page=1), dict(news=[1] * 300, lens=[i % 40 + 1 for i in range(300)], page=64),
         dict(news=[30] * 5, lens=[100] * 5, rank=64, q_rank=448), dict(news=[3], lens=[9], rank=8, q_rank=8)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", NORMS, ids=lambda c: "-".join(f"{k}{str(v)[:16]}" for k, v in c.items()))
def test_norms_match_float64_and_land_in_their_pages(case, dtype):
    from sophia_amd import ops
    case = dict(case)
    q_rank = case.pop("q_rank", 384)
    c = ref.Paged(**case, heads=1, dtype=dtype, behind=2)
    rank = c.pages.size(2)
    proj = torch.randn(c.rows, q_rank + rank + 16, generator=c.gen).to(dtype)
    q, kv = proj[:, :q_rank], proj[:, q_rank:q_rank + rank]
    q_w, kv_w = 1 + 0.1 * torch.randn(q_rank, generator=c.gen), 1 + 0.1 * torch.randn(rank, generator=c.gen)
    dev = proj.cuda()
    pages = c.pages.cuda()
    ops.mla_latent_norms_paged(dev[:, :q_rank], dev[:, q_rank:q_rank + rank], q_w.cuda(), 1e-5, kv_w.cuda(), 1e-6, pages,
                               *_dev(c.table, c.cu, c.kv_len), slots=c.slots.cuda())
    want = ref.norms(q, kv, q_w, 1e-5, kv_w, 1e-6)
    # the sum of up to 448 squares, a reciprocal root to 2 units, three products; then the result's rounding
    rel = (512 + 12) * E32 + (2.0 ** -8 if dtype == BF else E32)
    for got, w in zip((dev[:, :q_rank], dev[:, q_rank:q_rank + rank]), want):
        _within(got, w, rel * w.abs() + 1e-30)
    assert torch.equal(dev[:, q_rank + rank:].cpu(), proj[:, q_rank + rank:])
    expect, done = c.pages.clone(), dev[:, q_rank:q_rank + rank].cpu()
    for s, (n, length) in enumerate(zip(c.news, c.lens)):
        for i in range(n):
            expect[c.place(s, length - n + i)] = done[int(c.cu[s]) + i]
    assert torch.equal(pages.cpu().nan_to_num(9.0), expect.nan_to_num(9.0))


def test_norms_write_nothing_where_there_is_no_page():
    from sophia_amd import ops
    c = ref.Paged([6, 4, 3, 2, 1], [40, 20, 64, 9, 12], heads=1, spare=0)
    c.table[int(c.slots[0]), 2] = -1                 # positions 34 .. 39 have none
    c.kv_len[1] = 2                                   # two rows before position 0
    c.kv_len[2] = 66                                  # past the table
    c.slots[3] = 77
    c.table[int(c.slots[4]), 0] = c.pages.size(0)    # past the pool
    proj = torch.randn(c.rows, 512, generator=c.gen).to(BF).cuda()
    room = torch.full((c.pages.size(0) + 4, 16, 128), 5.0, dtype=BF, device="cuda")
    pool = room[2:-2]
    ops.mla_latent_norms_paged(proj[:, :384], proj[:, 384:], torch.ones(384).cuda(), 1e-5, torch.ones(128).cuda(), 1e-5, pool,
                               *_dev(c.table, c.cu, c.kv_len), slots=c.slots.cuda())
    done = proj[:, 384:].cpu()
    expect = torch.full(room.shape, 5.0, dtype=BF)
    page, _ = c.place(1, 0)
    expect[2 + page, 0], expect[2 + page, 1] = done[8], done[9]
    page, at = c.place(2, 63)
    expect[2 + page, at] = done[10]
    assert torch.equal(room.cpu(), expect)


# ------------------------------------------------------------------ beams
def _beam(logits, scores, beams, keep, ended=None, pad=3):
    from sophia_amd import ops
    got = ops.beam_select(*_dev(logits, scores), beams, keep=keep, ended=None if ended is None else ended.cuda(), pad_token=pad)
    want = ref.beam(logits, scores, beams, keep, ended, pad)
    assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu(), want[2])
    # sums of e^x to 2^-22 each, in fp32 of 32 values at most by themselves; the result's rounding
    some = want[1] >= 0
    err = (got[0].double().cpu() - want[0]).abs()
    assert bool((err[some] <= 2.0 ** -18 + E32 * want[0][some].abs()).all()), float(err[some].max())
    assert torch.equal(got[0].cpu()[~some], torch.full_like(got[0].cpu()[~some], float("-inf")))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("groups,beams,keep,vocab", [
    (1, 1, 1, 1), (1, 1, 4, 3), (2, 3, 7, 17), (1, 4, 8, 65536), (3, 2, 4, 2047), (2, 5, 10, 2049), (5, 8, 16, 5000), (1, 64, 64, 999),
    (2, 1, 64, 30000), (40, 4, 8, 32001), (150, 1, 2, 70000)])
def test_beams_match_float64(groups, beams, keep, vocab, dtype):
    gen = torch.Generator().manual_seed(groups + 7 * beams + vocab)
    rows = groups * beams
    logits = (torch.randn(rows, vocab, generator=gen) * 3).to(dtype)
    scores = -20 * torch.rand(rows, generator=gen)
    _beam(logits, scores, beams, keep)
    _beam(logits, scores, beams, keep, torch.rand(rows, generator=gen) < 0.4)


@pytest.mark.parametrize("groups,beams,keep,vocab", [(1, 1, 64, 65536), (2, 16, 64, 32008), (1, 16, 33, 40000), (2, 3, 48, 8200), (3, 12, 32, 32768)])
def test_beams_that_keep_many(groups, beams, keep, vocab):
    """Lists in one work-group's registers or more, parts that end within 8 values and not."""
    gen = torch.Generator().manual_seed(keep + vocab)
    logits = (torch.randn(groups * beams, vocab, generator=gen) * 3).to(BF)
    logits[:, ::7] = float("-inf")
    logits[0, 3::11] = float("nan")
    _beam(logits, -torch.rand(groups * beams, generator=gen), beams, keep)


@pytest.mark.parametrize("vocab", [1000, 9000, 40000])
def test_beams_equal_values_go_to_the_lowest(vocab):
    """Whole rows of one value, few different values, and equal beams: more equal candidates than any set holds."""
    gen = torch.Generator().manual_seed(vocab)
    for logits in (torch.zeros(4, vocab), torch.randint(0, 3, (4, vocab), generator=gen).float()):
        logits[2:] = logits[:2]
        _beam(logits, torch.tensor([-1.0, -2.0, -1.0, -2.0]), 2, 16)
    same = torch.randint(0, 3, (1, vocab), generator=gen).float().expand(4, vocab).contiguous()
    _beam(same, torch.full((4,), -1.0), 4, 64)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_beams_few_tokens_allowed_and_values_that_are_none(dtype):
    gen = torch.Generator().manual_seed(5)
    inf, nan, V = float("inf"), float("nan"), 30000
    logits = (torch.randn(12, V, generator=gen) * 2).to(dtype)
    logits[0, 3:] = -inf                    # three tokens
    logits[1] = -inf                        # none
    logits[2, 100:20000] = -inf             # some parts of the row without any, others whole
    logits[3, ::2] = nan
    logits[4] = nan
    logits[5, 77] = inf
    logits[6, 2500:] = -inf                 # more than fit, in one part
    scores = -torch.rand(12, generator=gen)
    scores[8], scores[9], scores[10] = -inf, nan, inf
    _beam(logits, scores, 1, 8)
    _beam(logits, scores, 4, 64)
    ended = torch.zeros(12, dtype=torch.bool)
    ended[[1, 4, 8, 10, 11]] = True
    _beam(logits, scores, 3, 5, ended)
    _beam(logits[1:2].contiguous(), torch.zeros(1), 1, 3)


def test_beams_strided_and_unaligned_logits():
    gen = torch.Generator().manual_seed(9)
    wide = torch.randn(6, 3001, generator=gen).to(BF)
    from sophia_amd import ops
    scores = -torch.rand(6, generator=gen)
    for cut in (wide[:, 1:], wide[:, 8:3000], wide[::2][:, :2999], wide[:, :2992]):
        rows = cut.size(0)
        dev = wide.cuda()
        view = dev[::2][:, :2999] if rows == 3 else dev[:, cut.storage_offset():cut.storage_offset() + cut.size(1)]
        got = ops.beam_select(view, scores[:rows].cuda(), 3, keep=9)
        want = ref.beam(cut, scores[:rows], 3, 9)
        assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu(), want[2])


# ------------------------------------------------------------------ moves
def _maps(kind, n, limit, rng):
    if kind == "random":
        return [rng.randrange(limit) for _ in range(n)], [rng.randrange(limit) for _ in range(n)]
    if kind == "distinct":
        return [rng.randrange(limit) for _ in range(n)], rng.sample(range(limit), n)
    if kind == "permutation":
        dst = rng.sample(range(limit), n)
        src = dst[:]
        rng.shuffle(src)
        return src, dst
    if kind == "rotation":
        return [(i + 1) % n for i in range(n)], list(range(n))
    if kind == "chain":
        return list(range(n)), [i + 1 for i in range(n)]
    if kind == "swaps":
        return [i ^ 1 for i in range(n)], list(range(n))
    src, dst = _maps("random", n, limit, rng)          # bad: slots that are none among the others
    for i in range(0, n, 3):
        (src if i % 2 else dst)[i] = rng.choice([-1, limit, limit + 7, 2 ** 31 - 1, -2 ** 31])
    return src, dst


KINDS = ["random", "distinct", "permutation", "rotation", "chain", "swaps", "bad"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,limit", [(1, 2), (2, 3), (4, 7), (31, 40), (64, 65), (300, 500), (1025, 1100), (4096, 4500)])
def test_page_copy_is_as_if_at_once(kind, n, limit):
    from sophia_amd import ops
    rng = random.Random(n * 31 + len(kind))
    n -= kind == "swaps" and n % 2
    src, dst = _maps(kind, n, limit, rng)
    pools = [torch.randn(limit, 4, 8).to(BF) for _ in range(2)]
    dev = _dev(*pools)
    ops.page_copy(*(torch.tensor(t, dtype=torch.int32).cuda() for t in (src, dst)), dev)
    for got, pool in zip(dev, pools):
        assert torch.equal(got.cpu(), ref.moved(pool, src, dst))


@pytest.mark.parametrize("dtype,page,rank", [(BF, 64, 128), (F32, 16, 256), (F32, 1, 8), (BF, 128, 40)])
def test_page_copy_moves_whole_pages_and_nothing_else(dtype, page, rank):
    from sophia_amd import ops
    both = torch.randn(30, 2, page, rank).to(dtype)
    dev = both.cuda()
    rng = random.Random(3)
    src, dst = _maps("distinct", 20, 30, rng)
    ops.page_copy(*(torch.tensor(t, dtype=torch.int32).cuda() for t in (src, dst)), [dev[:, 1]])
    assert torch.equal(dev[:, 0].cpu(), both[:, 0]) and torch.equal(dev[:, 1].cpu(), ref.moved(both[:, 1], src, dst))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,limit,width", [(1, 2, 6), (4, 5, 6), (9, 12, 6), (24, 30, 6), (64, 66, 40), (70, 90, 14)])
def test_fork_moves_every_cache(kind, n, limit, width):
    """Moves with tokens of their own each: a row of the table that moves is read for the pages of other moves."""
    from sophia_amd import ops
    rng = random.Random(n * 17 + len(kind))
    n -= kind == "swaps" and n % 2
    src, dst = _maps(kind, n, limit, rng)
    gen = torch.Generator().manual_seed(n)
    heads, page = 2, 16
    kda = [(torch.randn(limit, 3 * heads * 128, 3, generator=gen), torch.randn(limit, heads, 128, 128, generator=gen)) for _ in range(2)]
    mla = [torch.randn(limit, 90, 32, generator=gen) for _ in range(2)]
    table = torch.randperm(limit * width, generator=gen).view(limit, width).int()     # every slot's pages its own
    pools = [torch.randn(limit * width, page, 32, generator=gen).to(BF) for _ in range(2)]
    cached = torch.tensor([rng.choice([0, 1, 15, 16, 17, 40, 89, 96, 200, 600, -3]) for _ in range(n)], dtype=torch.int64)
    dk = [(c.cuda(), s.cuda()) for c, s in kda]
    dm, dp, dt = _dev(*mla), _dev(*pools), table.cuda()
    ops.cache_fork(*(torch.tensor(t, dtype=torch.int32).cuda() for t in (src, dst)), kda=dk, mla=dm, pools=dp, table=dt,
                   cached=cached.cuda())
    for (c, s), (gc, gs) in zip(kda, dk):
        assert torch.equal(gc.cpu(), ref.moved(c, src, dst)) and torch.equal(gs.cpu(), ref.moved(s, src, dst))
    for got, t in zip(dm, mla):
        assert torch.equal(got.cpu(), ref.fork_latents(t, src, dst, cached))
    want_table, want = ref.fork_pages(table, pools, src, dst, cached, limit)
    assert torch.equal(dt.cpu(), want_table)
    for got, w in zip(dp, want):
        assert torch.equal(got.cpu(), w)


def test_fork_of_parts_of_the_caches():
    """States without conv histories, latents alone, pages alone; no moves; pages that are none."""
    from sophia_amd import ops
    src, dst = (torch.tensor(t, dtype=torch.int32).cuda() for t in ([0, 0, 3], [1, 2, 0]))
    cached = torch.tensor([20, 20, 35], dtype=torch.int64).cuda()
    state = torch.randn(4, 1, 128, 128)
    dev = state.cuda()
    ops.cache_fork(src, dst, kda=[(None, dev)])
    assert torch.equal(dev.cpu(), ref.moved(state, [0, 0, 3], [1, 2, 0]))
    latents = torch.randn(4, 50, 64)
    dev = latents.cuda()
    ops.cache_fork(src, dst, mla=[dev], cached=cached)
    assert torch.equal(dev.cpu(), ref.fork_latents(latents, [0, 0, 3], [1, 2, 0], [20, 20, 35]))
    table = torch.arange(12).view(4, 3).int()
    table[1, 1], table[0, 2], table[2, 1] = -1, 99, 12
    pool = torch.randn(12, 16, 64)
    dt, dp = table.cuda(), pool.cuda()
    ops.cache_fork(src, dst, pools=[dp], table=dt, cached=cached)
    want_table, want = ref.fork_pages(table, [pool], [0, 0, 3], [1, 2, 0], [20, 20, 35], 4)
    assert torch.equal(dt.cpu(), want_table) and torch.equal(dp.cpu(), want[0])
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.cache_fork(none, none, kda=[(None, dev)])
    ops.cache_fork(src, dst)
    ops.page_copy(none, none, [dp])
    assert torch.equal(dp.cpu(), want[0])
