"""The kernels for what single requests ask of a batch: low-rank adapters, changes of logits, log-probabilities."""
import math
import random

import pytest
import torch

import request_cases as rc

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def ops():
    from ninfer_amd.kernels import load_ops
    return load_ops()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def f32(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


# ---- adapters --------------------------------------------------------------------------------------

def tables(count, k, widths, r, dtype, seed, x_rows):
    gen = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    return (rand(x_rows, k).to(dtype), (rand(count, len(widths) * r, k) * k ** -0.5).to(dtype), rand(count, sum(widths), r).to(dtype),
            torch.rand(count, generator=gen, device="cuda") * 2 - 0.5, rand(x_rows, sum(widths)).to(dtype))


def rows_of(kind, t, count, rng):
    if kind == "one":
        return [count - 1] * t
    if kind == "none":
        return [-1] * t
    if kind == "mixed":     # every row its own, also numbers that name no adapter
        return [rng.choice([-1, count, 2 ** 31 - 1, -2 ** 31] + list(range(count)) * 3) for _ in range(t)]
    rows = []               # portions
    while len(rows) < t:
        rows += [rng.randrange(-1, count)] * rng.randint(1, 40)
    return rows[:t]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k,widths,r,count", [
    (1, 64, (64,), 16, 1), (1, 2048, (256, 64, 64), 16, 4), (2, 1, (1,), 1, 2), (3, 33, (7, 5, 1, 2), 3, 3),
    (15, 96, (48,), 8, 5), (16, 128, (64, 32, 32), 32, 16), (17, 1000, (100, 60), 24, 7), (64, 512, (192, 64), 64, 8),
    (65, 257, (65, 63, 64), 20, 3), (130, 320, (130,), 40, 2), (700, 264, (72, 8, 16), 12, 6), (33, 72, (16,), 129, 4), (9, 72, (16, 600), 100, 4), (16, 2048, (1100, 70), 64, 16), (16, 2048, (1100, 70), 16, 16), (11, 1030, (513, 9, 30, 64), 13, 40)])
@pytest.mark.parametrize("kind", ["one", "mixed", "portions"])
def test_adapters(ops, dtype, t, k, widths, r, count, kind):
    rng = random.Random(t * 7 + k)
    x, a, b, scale, base = tables(count, k, widths, r, dtype, t + k, t)
    ranks = [rng.choice((r, max(1, r // 2), rng.randint(0, r))) for _ in range(count)]
    ranks[-1] = r
    rows = i32(rows_of(kind, t, count, rng))
    want, room = rc.adapters(x, a, b, scale, ranks, widths, rows, base)
    out = torch.full_like(base, NAN)
    kept = base.clone()
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, rows, out, base=base)
    rc.close(out, want, room)
    assert torch.equal(base, kept)
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, rows, base)   # in place: the same bits
    assert torch.equal(base, out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,count", [(512, 1), (600, 70), (1537, 9), (2061, 40), (6200, 3)])
@pytest.mark.parametrize("kind", ["one", "mixed", "portions", "last"])
def test_adapters_of_many_rows(ops, dtype, t, count, kind):
    """Tiles of one adapter, of as many as rows, and a step of which only the last rows have any."""
    k, widths, r = 136, (80, 24), 8
    rng = random.Random(t)
    x, a, b, scale, base = tables(count, k, widths, r, dtype, t, t)
    ranks = [rng.randint(0, r) for _ in range(count)]
    ranks[-1] = r
    rows = [-1] * (t - 9) + [i % count for i in range(9)] if kind == "last" else rows_of(kind, t, count, rng)
    want, room = rc.adapters(x.cpu(), a.cpu(), b.cpu(), scale.cpu(), ranks, widths, torch.tensor(rows), base.cpu())
    out = torch.full_like(base, NAN)
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, i32(rows), out, base=base)
    rc.close(out, want, room)
    split = torch.full_like(base, NAN)
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, i32(rows), split, base=base, single_rows=37)   # the same bits
    assert torch.equal(split, out)
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, i32(rows), base)
    assert torch.equal(base, out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k,r,count", [(600, 136, 8, 9), (640, 129, 13, 40), (1100, 72, 64, 1), (577, 200, 80, 70)])
@pytest.mark.parametrize("kind", ["one", "mixed", "portions", "singles"])
def test_adapters_of_many_columns(ops, dtype, t, k, r, count, kind):
    """Enough columns for tiles of 32 rows in the second product, whatever the first one's are."""
    widths, rng = (1500, 77, 1000), random.Random(t)
    x, a, b, scale, base = tables(count, k, widths, r, dtype, t, t)
    ranks = [rng.randint(0, r) for _ in range(count)]
    ranks[-1] = r
    rows = [i % count for i in range(30)] + [0] * (t - 30) if kind == "singles" else rows_of(kind, t, count, rng)
    want, room = rc.adapters(x.cpu(), a.cpu(), b.cpu(), scale.cpu(), ranks, widths, torch.tensor(rows), base.cpu())
    out = torch.full_like(base, NAN)
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, i32(rows), out, base=base)
    rc.close(out, want, room)
    for single in (15, 30, t):   # (the same bits: what is said of the rows changes the time alone)
        again = torch.full_like(base, NAN)
        ops.adapter_add(x, a, b, scale, i32(ranks), widths, i32(rows), again, base=base, single_rows=single)
        assert torch.equal(again, out)
    some = list(range(0, 8)) + list(range(t - 8, t))
    got = torch.empty_like(base[some])
    ops.adapter_add(x[some], a, b, scale, i32(ranks), widths, i32([rows[i] for i in some]), got, base=base[some])
    assert torch.equal(got, out[some])


def test_adapters_rows_without_one_keep_their_bits(ops):
    x, a, b, scale, base = tables(3, 128, (64, 64), 16, torch.bfloat16, 1, 40)
    base[3, 5], base[7, 9] = NAN, INF
    a[:] = NAN
    before = base.clone()
    for rows in (rows_of("none", 40, 3, None), [3, -5] * 20):
        ops.adapter_add(x, a, b, scale, i32([16, 16, 16]), (64, 64), i32(rows), base)
        out = torch.zeros_like(base)
        ops.adapter_add(x, a, b, scale, i32([16, 16, 16]), (64, 64), i32(rows), out, base=base)
        for got in (base, out):
            assert torch.equal(got.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_adapters_read_nothing_beyond_a_rank_and_mix_no_rows(ops, dtype):
    t, k, widths, r, count = 48, 256, (96, 32), 24, 4
    x, a, b, scale, base = tables(count, k, widths, r, dtype, 3, t)
    ranks, rows = [24, 5, 0, 11], [(i * 7) % 5 - 1 for i in range(t)]
    for g, rank in enumerate(ranks):
        b[g, :, rank:] = NAN
        for s in range(2):
            a[g, s * r + rank:(s + 1) * r] = NAN
    x[5], x[17], x[20, 3] = NAN, INF, NAN
    sick = [i for i in (5, 17, 20) if rows[i] >= 0 and ranks[rows[i]] > 0]
    assert sick
    out = torch.empty_like(base)
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, i32(rows), out, base=base)
    fine = [i for i in range(t) if i not in sick]
    want, room = rc.adapters(x[fine], a, b, scale, ranks, widths, i32([rows[i] for i in fine]), base[fine])
    rc.close(out[fine], want, room)
    assert not torch.isfinite(out[sick]).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_adapters_on_columns_of_wider_rows(ops, dtype, shift):
    t, k, widths, r, count = 37, 128, (64, 32), 16, 3
    x, a, b, scale, base = tables(count, k, widths, r, dtype, shift, t)
    rows, ranks = i32([i % 4 - 1 for i in range(t)]), [16, 9, 16]
    wide_x = torch.full((t, k + 11), NAN, dtype=dtype, device="cuda")
    wide_x[:, shift:shift + k] = x
    wide = torch.full((t, 96 + 13), 7.0, dtype=dtype, device="cuda")
    wide[:, shift:shift + 96] = base
    want, room = rc.adapters(x, a, b, scale, ranks, widths, rows, base)
    ops.adapter_add(wide_x[:, shift:shift + k], a, b, scale, i32(ranks), widths, rows, wide[:, shift:shift + 96])
    rc.close(wide[:, shift:shift + 96], want, room)
    assert (wide[:, :shift] == 7).all() and (wide[:, shift + 96:] == 7).all()


def test_adapters_give_a_row_the_same_bits_in_any_company(ops):
    t, k, widths, r, count = 640, 512, (256, 128, 128), 64, 8
    x, a, b, scale, base = tables(count, k, widths, r, torch.bfloat16, 9, t)
    ranks = i32([64, 16, 33, 64, 8, 1, 64, 40])
    rows = [i % 9 - 1 for i in range(t)]
    out = torch.empty_like(base)
    ops.adapter_add(x, a, b, scale, ranks, widths, i32(rows), out, base=base)
    for some in ([0], [5], list(range(100, 116)), list(range(3, 640, 11)), list(range(128, 400))):
        got = torch.empty_like(base[some])
        ops.adapter_add(x[some], a, b, scale, ranks, widths, i32([rows[i] for i in some]), got, base=base[some])
        assert torch.equal(got, out[some])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_adapters_of_small_rank_give_a_row_the_same_bits_in_any_company(ops, dtype):
    # (16 rows go through one launch, more through two)
    t, k, widths, r, count = 50, 1000, (600, 64), 16, 6
    x, a, b, scale, base = tables(count, k, widths, r, dtype, 10, t)
    ranks, rows = i32([16, 3, 16, 0, 9, 16]), [i * 5 % 7 - 1 for i in range(t)]
    out = torch.empty_like(base)
    ops.adapter_add(x, a, b, scale, ranks, widths, i32(rows), out, base=base)
    for some in ([0], [5], list(range(16)), list(range(30, 39)), list(range(3, 50, 4))):
        got = torch.empty_like(base[some])
        ops.adapter_add(x[some], a, b, scale, ranks, widths, i32([rows[i] for i in some]), got, base=base[some])
        assert torch.equal(got, out[some])


def test_adapters_beyond_32_bits(ops):
    # factors of more than 2^32 bytes, rows whose offsets pass 2^31 numbers
    k, n, r, count = 4096, 4096, 128, 2200
    a = torch.zeros(count, r, k, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(count, n, r, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator("cuda").manual_seed(0)
    for g in (0, count - 1):
        a[g] = torch.randn(r, k, generator=gen, device="cuda") / 64
        b[g] = torch.randn(n, r, generator=gen, device="cuda")
    x = torch.randn(4, k, generator=gen, device="cuda").bfloat16()
    base = torch.randn(4, n, generator=gen, device="cuda").bfloat16()
    rows, scale, ranks = i32([count - 1, 0, -1, count - 1]), torch.ones(count, device="cuda"), torch.full((count,), r, device="cuda").int()
    want, room = rc.adapters(x, a, b, scale, ranks, (n,), rows, base)
    ops.adapter_add(x, a, b, scale, ranks, (n,), rows, base)
    rc.close(base, want, room)
    del a, b
    stride = 1 << 30   # a row every 2^30 numbers
    room_for = torch.zeros(3 * stride + n, dtype=torch.bfloat16, device="cuda")
    out = room_for.as_strided((4, n), (stride, 1))
    a, b = (torch.randn(1, r, k, generator=gen, device="cuda") / 64).bfloat16(), torch.randn(1, n, r, generator=gen, device="cuda").bfloat16()
    want, room = rc.adapters(x, a, b, scale, [r], (n,), i32([0, 0, -1, 0]), torch.zeros(4, n, dtype=torch.bfloat16, device="cuda"))
    ops.adapter_add(x, a, b, scale[:1], i32([r]), (n,), i32([0, 0, -1, 0]), out)
    rc.close(out, want, room)


def test_adapters_refusals(ops):
    from ninfer_amd.kernels.ops import KernelError
    x, a, b, scale, base = tables(2, 64, (32, 32), 8, torch.bfloat16, 0, 4)
    ranks, rows = i32([8, 8]), i32([0, 1, -1, 0])
    before = base.clone()
    bad = [dict(x=x.float()), dict(x=x[:, :63]), dict(a=a[:, :15]), dict(b=b[:, :, :7]), dict(scale=scale.double()),
           dict(scale=scale[:1]), dict(ranks=ranks.long()), dict(rows=rows[:3]), dict(widths=(32, 31)), dict(widths=(64,)),
           dict(widths=(64, 0)), dict(widths=()), dict(out=base[:3]), dict(out=base.float()), dict(x=x.cpu()), dict(out=base.t()),
           dict(base=base.float()), dict(x=x[:1].expand(4, 64)), dict(out=base[:1].expand(4, 64)), dict(a=a.cpu())]
    for change in bad:
        c = dict(dict(x=x, a=a, b=b, scale=scale, ranks=ranks, widths=(32, 32), rows=rows, out=base, base=None), **change)
        with pytest.raises(KernelError):
            ops.adapter_add(c["x"], c["a"], c["b"], c["scale"], c["ranks"], c["widths"], c["rows"], c["out"], base=c["base"])
    wide = torch.zeros(5, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError, match="overlap"):
        ops.adapter_add(x, a, b, scale, ranks, (32, 32), rows, wide[1:], base=wide[:4])
    with pytest.raises(KernelError, match="overlap"):
        ops.adapter_add(x, a, b, scale, ranks, (32, 32), rows, x)
    for single in (-1, 5):
        with pytest.raises(KernelError, match="single rows"):
            ops.adapter_add(x, a, b, scale, ranks, (32, 32), rows, base, single_rows=single)
    with pytest.raises(KernelError, match="together"), ops.together():
        ops.adapter_add(x, a, b, scale, ranks, (32, 32), rows, base)
    assert torch.equal(base, before)
    ops.adapter_add(x[:0], a, b, scale, ranks, (32, 32), rows[:0], base[:0])   # no rows: nothing to do


# ---- changes of logits -----------------------------------------------------------------------------

def make_adjust(rows, vocab, seed, history=True, biases=True, masks=True):
    rng = random.Random(seed)
    token = lambda: rng.choice([rng.randrange(vocab), rng.randrange(min(vocab, 50)), vocab - 1, 0])
    c = dict(repetition=[rng.choice((1.0, 0.7, 1.3, 2.0)) for _ in range(rows)], presence=[rng.uniform(-2, 2) for _ in range(rows)],
             frequency=[rng.choice((0.0, rng.uniform(-1, 1))) for _ in range(rows)])
    # (the same token more than once, ids outside the vocabulary, rows with nothing)
    c["histories"] = [[(rng.choice((token(), token(), token(), vocab, -1, 2 ** 31 - 1, -2 ** 31)), n, rng.randint(0, n))
                       for n in [rng.choice((1, 2, 5, 40)) for _ in range(rng.choice((0, 1, 30, 600)))]] for _ in range(rows)]
    c["biases"] = [[(rng.choice((token(), token(), token(), vocab, -9)), rng.choice((rng.uniform(-9, 9), -INF, INF, -100.0)))
                    for _ in range(rng.choice((0, 2, 70)))] for _ in range(rows)]
    c["masks"] = [[rng.random() < 0.5 for _ in range(vocab)], [False] * vocab, [True] * vocab]
    c["mask_rows"] = [rng.choice((-1, 0, 1, 2, 3, 2 ** 31 - 1)) for _ in range(rows)]
    if not history:
        c["histories"] = None
    if not biases:
        c["biases"] = None
    if not masks:
        c["masks"] = c["mask_rows"] = None
    return c


def on_gpu(c):
    kw = dict(repetition=f32(c["repetition"]), presence=f32(c["presence"]), frequency=f32(c["frequency"]))
    if c["histories"] is not None:
        offsets, cols = rc.lists(c["histories"])
        cols = cols or [[], [], []]
        kw.update(hist_offsets=i32(offsets), hist_tokens=i32(cols[0]), hist_counts=i32(cols[1]), hist_generated=i32(cols[2]))
    if c["biases"] is not None:
        offsets, cols = rc.lists(c["biases"])
        cols = cols or [[], []]
        kw.update(bias_offsets=i32(offsets), bias_tokens=i32(cols[0]), bias_values=f32(cols[1]))
    if c["masks"] is not None:
        kw.update(masks=i32([rc.pack(m) for m in c["masks"]]), mask_rows=i32(c["mask_rows"]))
    return kw


def rounded(c):
    """The 32-bit numbers that the kernel is given."""
    c = dict(c)
    for k in ("repetition", "presence", "frequency"):
        c[k] = torch.tensor(c[k], dtype=torch.float32)
    if c["biases"] is not None:
        c["biases"] = [[(t, float(torch.tensor(v, dtype=torch.float32))) for t, v in r] for r in c["biases"]]
    return c


@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 31), (3, 32), (1, 33), (5, 1000), (4, 4095), (3, 4096), (2, 4097), (7, 9001), (2, 151936)])
@pytest.mark.parametrize("what", ["all", "history", "biases", "masks", "nothing"])
def test_adjust(ops, rows, vocab, what):
    c = make_adjust(rows, vocab, rows * vocab, what in ("all", "history"), what in ("all", "biases"), what in ("all", "masks"))
    logits = 3 * torch.randn(rows, vocab, generator=torch.Generator("cuda").manual_seed(vocab), device="cuda")
    if vocab > 30:   # NaN and infinities, where a mask may bar them and where none does
        logits[0, 3], logits[-1, 7], logits[0, 11], logits[0, 5] = NAN, INF, -INF, 0.0
    want, room = rc.adjusted(logits, **rounded(c))
    out, kept = torch.full_like(logits, NAN), logits.clone()
    kw = on_gpu(c)
    ops.adjust_logits(logits, out, **kw)
    rc.close(out, want, room)
    assert torch.equal(logits.view(torch.int32), kept.view(torch.int32))
    ops.adjust_logits(logits, **kw)   # in place: the same bits
    assert torch.equal(logits.view(torch.int32), out.view(torch.int32))


@pytest.mark.parametrize("shift,pad", [(0, 4), (1, 6), (4, 4), (2, 3)])
def test_adjust_rows_of_wider_ones(ops, shift, pad):
    rows, vocab = 5, 5003
    c = make_adjust(rows, vocab, 3)
    wide = torch.randn(rows, vocab + shift + pad, device="cuda")
    kept = wide.clone()
    want, room = rc.adjusted(wide[:, shift:shift + vocab], **rounded(c))
    ops.adjust_logits(wide[:, shift:shift + vocab], **on_gpu(c))
    rc.close(wide[:, shift:shift + vocab], want, room)
    assert torch.equal(wide[:, :shift], kept[:, :shift]) and torch.equal(wide[:, shift + vocab:], kept[:, shift + vocab:])


def test_adjust_counts_of_any_size(ops):
    logits = f32([[2.0, -2.0, 0.0, 1e30, -1e30, 3.0, INF, -INF]])
    counts = [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 300, 300, 70000, 90000, 90000]
    for p in (1.5, 0.5, 1.0 + 2.0 ** -23, 1.0000001192092896):
        c = dict(repetition=[p], presence=[0.5], frequency=[0.0], histories=[[(t, n, 0) for t, n in enumerate(counts)]],
                 biases=None, masks=None, mask_rows=None)
        want, room = rc.adjusted(logits, **rounded(c))
        out = torch.empty_like(logits)
        ops.adjust_logits(logits, out, **on_gpu(c))
        # (a power of so many squarings in 64 bits is off by the count times 2^-52, beyond 32 bits' step only for such counts)
        much = want.abs() * torch.tensor(counts).double() * 2.0 ** -52
        rc.close(out, want, room + torch.nan_to_num(much, posinf=0, neginf=0) + 2.0 ** -149)


def test_adjust_without_a_history_of_generated_tokens(ops):
    logits = torch.randn(2, 100, device="cuda")
    out = torch.empty_like(logits)
    ops.adjust_logits(logits, out, repetition=f32([2.0, 1.0]), presence=f32([1.0, 1.0]), hist_offsets=i32([0, 1, 2]),
                      hist_tokens=i32([4, 4]), hist_counts=i32([1, 1]))
    want = logits.clone()
    want[0, 4] = want[0, 4] / 2 if want[0, 4] > 0 else want[0, 4] * 2
    assert torch.equal(out, want)


def test_adjust_offsets_that_leave_the_lists_read_nothing(ops):
    logits = torch.randn(3, 64, device="cuda")
    out = torch.empty_like(logits)
    ops.adjust_logits(logits, out, presence=f32([9.0] * 3), hist_offsets=i32([-5, 1, 2 ** 31 - 1, 2]), hist_tokens=i32([1, 2]),
                      hist_counts=i32([1, 1]), hist_generated=i32([1, 1]))
    want = logits.clone()
    want[0, 1] -= 9
    want[1, 2] -= 9
    assert torch.equal(out, want)


@pytest.mark.parametrize("vocab", [4092, 4093, 4096, 9000])
def test_adjust_lists_of_every_token(ops, vocab):
    rows = 2
    c = make_adjust(rows, vocab, 5)
    order = random.Random(1).sample(range(vocab), vocab)
    c["histories"] = [[(t, 1 + t % 3, t % 2) for t in order], []]
    c["biases"] = [[], [(t, float(t % 17)) for t in order]]
    logits = torch.randn(rows, vocab, device="cuda")
    want, room = rc.adjusted(logits, **rounded(c))
    ops.adjust_logits(logits, **on_gpu(c))
    rc.close(logits, want, room)


@pytest.mark.parametrize("biases", [63, 64, 65, 130])
def test_adjust_biases_of_one_part(ops, biases):
    rng = random.Random(biases)
    c = dict(repetition=[1.5], presence=[0.25], frequency=[0.5], histories=[[(t, 1 + t % 3, t % 2) for t in range(0, 90, 2)]],
             biases=[[(rng.randrange(90), rng.uniform(-4, 4)) for _ in range(biases)]], masks=None, mask_rows=None)
    logits = torch.randn(1, 4096, generator=torch.Generator("cuda").manual_seed(biases), device="cuda")
    want, room = rc.adjusted(logits, **rounded(c))
    ops.adjust_logits(logits, **on_gpu(c))
    rc.close(logits, want, room)


@pytest.mark.parametrize("which", ["histories", "biases", "both"])
def test_adjust_lists_of_a_million_entries(ops, which):
    rng, n, vocab = random.Random(3), (1 << 20) + 77, 5001
    ids = [rng.randrange(-50, vocab + 50) for _ in range(n)]
    few = [(t, 1, 1) for t in (0, 7, 4999)], [(t, 0.5) for t in (1, 7, 4999)]
    c = dict(repetition=[1.0 + 2.0 ** -10], presence=[0.25], frequency=[2.0 ** -9], masks=None, mask_rows=None,
             histories=[[(t, 1, i % 2) for i, t in enumerate(ids)] if which != "biases" else few[0]],
             biases=[[(t, (i % 64) / 8) for i, t in enumerate(ids)] if which != "histories" else few[1]])
    logits = torch.randn(1, vocab, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    want, room = rc.adjusted(logits, **rounded(c))
    ops.adjust_logits(logits, **on_gpu(c))
    rc.close(logits, want, room)


def test_adjust_refusals(ops):
    from ninfer_amd.kernels.ops import KernelError
    logits, one = torch.zeros(2, 64, device="cuda"), f32([1.0, 1.0])
    offsets, tokens = i32([0, 1, 2]), i32([1, 2])
    words = i32([[0, 0]])
    for args, kw in [
            ((logits.bfloat16(),), {}), ((logits.cpu(),), {}), ((logits, logits[:1]), {}), ((logits, logits.t()), {}),
            ((logits,), dict(repetition=one[:1])), ((logits,), dict(presence=one.double())), ((logits,), dict(frequency=one.cpu())),
            ((logits,), dict(hist_offsets=offsets, hist_tokens=tokens)), ((logits,), dict(hist_offsets=offsets[:2], hist_tokens=tokens, hist_counts=tokens)),
            ((logits,), dict(hist_offsets=offsets, hist_tokens=tokens, hist_counts=tokens[:1])), ((logits,), dict(hist_generated=tokens)),
            ((logits,), dict(bias_offsets=offsets, bias_tokens=tokens)), ((logits,), dict(bias_offsets=offsets, bias_tokens=tokens, bias_values=tokens)),
            ((logits,), dict(masks=words)), ((logits,), dict(mask_rows=tokens)), ((logits,), dict(masks=i32([[0]]), mask_rows=tokens)),
            ((logits,), dict(masks=words.long(), mask_rows=tokens)), ((logits[:1].expand(2, 64),), {})]:
        with pytest.raises(KernelError):
            ops.adjust_logits(*args, **kw)
    wide = torch.zeros(3, 64, device="cuda")
    with pytest.raises(KernelError, match="overlap"):
        ops.adjust_logits(wide[:2], wide[1:])
    assert not logits.any()
    ops.adjust_logits(logits[:0], repetition=one[:0])


# ---- log-probabilities -----------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (2, 2, 1), (3, 63, 63), (2, 64, 64), (4, 300, 20), (1, 1000, 0), (5, 4096, 5), (3, 4097, 32),
                                            (2, 8191, 64), (9, 32001, 8), (2, 151936, 20), (70, 5000, 3)])
@pytest.mark.parametrize("kind", ["plain", "coarse", "sorted", "falling", "equal", "barred"])
def test_logprobs(ops, rows, vocab, top, kind):
    gen = torch.Generator("cuda").manual_seed(rows + vocab)
    logits = 4 * torch.randn(rows, vocab, generator=gen, device="cuda")
    if kind == "coarse":
        logits = logits.bfloat16().float()
    elif kind in ("sorted", "falling"):
        logits = torch.sort(logits, dim=1, descending=kind == "falling").values
    elif kind == "equal":
        logits = logits[:, :1].expand(rows, vocab).contiguous()
    elif kind == "barred":    # few tokens, fewer than are listed, have mass
        keep = torch.rand(rows, vocab, generator=gen, device="cuda") < min(0.5, 10 / vocab)
        keep[:, vocab // 2] = True
        logits = logits.masked_fill(~keep, -INF)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda").int()
    tokens[0] = int(logits[0].argmax())
    (p, before, best, bp), (room, broom) = rc.logprobs(logits, tokens, top)
    got = ops.token_logprobs(logits, tokens, top)
    rc.close(got[0], p, room)
    assert got[1].tolist() == before.tolist()
    assert got[2].tolist() == best.tolist()
    rc.close(got[3], bp, broom)
    if top:
        alone = ops.token_logprobs(logits, top=top)
        assert alone[0] is None and alone[1] is None
        assert torch.equal(alone[2], got[2]) and torch.equal(alone[3], got[3])
    assert torch.equal(ops.token_logprobs(logits, tokens)[0], got[0])   # without the list: the same bits
    assert torch.equal(ops.token_logprobs(logits[-1:], tokens[-1:], top)[3], got[3][-1:])   # ... and alone


def test_logprobs_of_infinities_and_nan(ops):
    x = torch.randn(6, 5000, device="cuda")
    x[0] = -INF
    x[1, 7] = x[1, 4999] = INF
    x[2, 4500] = NAN
    x[3] = NAN
    x[4, 10], x[4, 20] = -0.0, 0.0
    x[4, x[4] > 0] = -1.0
    x[5, :] = -INF
    x[5, 4321] = -3e38
    tokens = i32([5, 7, 3, 4, 20, 4321])
    p, before, best, bp = (v.tolist() for v in ops.token_logprobs(x, tokens, 3))
    assert p[0] == -INF and before[0] == 5 and best[0] == [0, 1, 2] and bp[0] == [-INF] * 3
    assert p[1] == pytest.approx(-math.log(2), abs=2 ** -23) and best[1][:2] == [7, 4999] and bp[1][2] == -INF and before[1] == 0
    assert math.isnan(p[2]) and 4500 not in best[2] and all(math.isnan(v) for v in bp[2])
    assert before[2] == int((x[2] > x[2, 3]).sum())
    assert math.isnan(p[3]) and before[3] == 4 and best[3] == [0, 1, 2]
    assert best[4][:2] == [10, 20] and before[4] == 1
    assert p[5] == 0.0 and best[5] == [4321, 0, 1] and bp[5] == [0.0, -INF, -INF]


def test_logprobs_of_a_row_with_many_nan(ops):
    # whole threads' logits and whole groups of them are NaN, and fewer than `top` are not
    x = torch.full((3, 9000), NAN, device="cuda")
    x[0, 100:120] = torch.arange(20.0)
    x[1, ::64] = torch.randn(141, device="cuda")
    x[2, 4096:] = torch.randn(4904, device="cuda")
    p, before, best, _ = ops.token_logprobs(x, i32([119, 64, 5000]), 40)
    for r in range(3):
        key = torch.where(x[r].isnan(), torch.full_like(x[r], -INF), x[r]).cpu()
        assert best[r].tolist() == torch.sort(key, descending=True, stable=True).indices[:40].tolist()
    assert before[0] == 0 and p.isnan().all()


@pytest.mark.parametrize("shift,pad", [(0, 3), (1, 3), (4, 4)])
def test_logprobs_rows_of_wider_ones_and_tokens_outside(ops, shift, pad):
    wide = torch.full((4, 6001 + shift + pad), 99.0, device="cuda")
    wide[:, shift:shift + 6001] = torch.randn(4, 6001, device="cuda")
    rows = wide[:, shift:shift + 6001]
    tokens = i32([6000, 0, 1, 2])
    (p, before, best, bp), (room, broom) = rc.logprobs(rows, tokens, 10)
    got = ops.token_logprobs(rows, tokens, 10)
    rc.close(got[0], p, room)
    rc.close(got[3], bp, broom)
    assert got[1].tolist() == before.tolist() and got[2].tolist() == best.tolist()
    got = ops.token_logprobs(rows, i32([-1, 6001, 2 ** 31 - 1, -2 ** 31]))
    assert all(math.isnan(v) for v in got[0].tolist()) and got[1].tolist() == [-1] * 4


def test_rows_of_logits_beyond_32_bits(ops):
    # a row every 2^30 numbers: the third lies behind 2^31 numbers, 2^33 bytes
    stride, vocab = 1 << 30, 5000
    rows = torch.zeros(2 * stride + vocab, device="cuda").as_strided((3, vocab), (stride, 1))
    rows.copy_(torch.randn(3, vocab, device="cuda"))
    tokens = i32([1, 2, 3])
    (p, before, best, bp), (room, broom) = rc.logprobs(rows, tokens, 4)
    got = ops.token_logprobs(rows, tokens, 4)
    rc.close(got[0], p, room)
    assert got[1].tolist() == before.tolist() and got[2].tolist() == best.tolist()
    c = make_adjust(3, vocab, 1)
    want, room = rc.adjusted(rows, **rounded(c))
    ops.adjust_logits(rows, **on_gpu(c))
    rc.close(rows, want, room)


def test_no_rows_and_no_tokens(ops):
    none = torch.zeros(0, 100, device="cuda")
    p, before, best, best_p = ops.token_logprobs(none, i32([]), 3)
    assert p.shape == before.shape == (0,) and best.shape == best_p.shape == (0, 3)
    ops.adjust_logits(none)
    p, before, best, best_p = ops.token_logprobs(torch.zeros(2, 0, device="cuda"), i32([0, 5]))
    assert p.isnan().all() and before.tolist() == [-1, -1] and best.shape == (2, 0)
    ops.adjust_logits(torch.zeros(2, 0, device="cuda"))


def test_logprobs_refusals(ops):
    from ninfer_amd.kernels.ops import KernelError
    x = torch.zeros(2, 50, device="cuda")
    for args in [(x.double(), None, 1), (x.cpu(), None, 1), (x, i32([1]), 1), (x, i32([1, 2]).long(), 1), (x, None, 51), (x, None, -1),
                 (torch.zeros(2, 100, device="cuda"), None, 65), (x.t(), None, 1), (x[:1].expand(2, 50), None, 1)]:
        with pytest.raises(KernelError):
            ops.token_logprobs(*args)
    got = ops.token_logprobs(x[:0], i32([]), 3)
    assert got[0].shape == (0,) and got[2].shape == (0, 3)


# ---- streams and graphs ----------------------------------------------------------------------------

def test_two_captured_graphs_and_another_stream(ops):
    """The three calls captured twice, replayed in turn and beside eager work on other inputs; then on a stream of their own."""
    t, k, widths, r, count, vocab = 24, 256, (64, 64), 16, 4, 5000
    sets = []
    for seed in (1, 2):
        x, a, b, scale, base = tables(count, k, widths, r, torch.bfloat16, seed, t)
        c = make_adjust(t, vocab, seed)
        sets.append(dict(x=x, a=a, b=b, scale=scale, base=base, ranks=i32([16, 3, 16, 8]), rows=i32([(i * seed) % 5 - 1 for i in range(t)]),
                         logits=torch.randn(t, vocab, device="cuda"), tokens=i32([(i * 37) % vocab for i in range(t)]), kw=on_gpu(c)))

    def run(s):
        out, changed = torch.empty_like(s["base"]), torch.empty_like(s["logits"])
        ops.adapter_add(s["x"], s["a"], s["b"], s["scale"], s["ranks"], widths, s["rows"], out, base=s["base"])
        ops.adjust_logits(s["logits"], changed, **s["kw"])
        return (out, changed) + ops.token_logprobs(changed, s["tokens"], 7)

    def check(got, s):
        for g, w in zip(got, run(s)):
            assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(w))

    run(sets[0])
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["out"] = run(s)
        graphs.append(g)
    for turn in range(3):
        for g, s in zip(graphs, sets):
            s["x"].normal_()
            s["logits"].normal_()
            s["rows"].copy_(torch.randint(-1, count, (t,), device="cuda"))
            g.replay()
        run(sets[turn % 2])   # eager work of the same sizes between them
        torch.cuda.synchronize()
        for s in sets:
            check(s["out"], s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run(s) for s in sets]
    side.synchronize()
    for g, s in zip(got, sets):
        check(g, s)


def test_the_sequence_of_a_step(ops):
    """A projection with adapters, its rows as logits, changed and read back: as a step of decoding requests uses them."""
    t, k, vocab, r = 8, 128, 3001, 8
    x, a, b, scale, _ = tables(3, k, (vocab,), r, torch.float32, 4, t)
    w = torch.randn(vocab, k, device="cuda") / 8
    rows, ranks = i32([0, 1, 2, -1, 0, 1, 2, -1]), [8, 8, 4]
    logits = torch.empty(t, vocab, device="cuda")
    ops.linear(x, w, logits)
    want, room = rc.adapters(x, a, b, scale, ranks, (vocab,), rows, logits)
    ops.adapter_add(x, a, b, scale, i32(ranks), (vocab,), rows, logits)
    rc.close(logits, want, room)
    c = make_adjust(t, vocab, 8)
    want, room = rc.adjusted(logits, **rounded(c))
    changed = torch.empty_like(logits)
    ops.adjust_logits(logits, changed, **on_gpu(c))
    rc.close(changed, want, room)
    tokens = torch.empty(t, dtype=torch.int32, device="cuda")
    ops.sample(changed, f32([0.0] * t), f32([0.0] * t), tokens)
    p, before, best, bp = ops.token_logprobs(logits, tokens, 4)
    (p64, before64, best64, bp64), (room, broom) = rc.logprobs(logits, tokens, 4)
    rc.close(p, p64, room)
    rc.close(bp, bp64, broom)
    assert before.tolist() == before64.tolist() and best.tolist() == best64.tolist()
