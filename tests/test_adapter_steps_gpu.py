"""Steps in which some requests have a low-rank adapter: what the others keep."""
import numpy as np
import pytest
import torch

import request_cases as rc
import util
from test_request_ops_gpu import i32, tables
from test_requests_gpu import adapters_of, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ninfer_amd.kernels import load_ops
    return load_ops()


def turned_case(t, k, heads, kv, d, r, count, dtype, seed):
    """Rows, weights, adapters and the cache of a projection whose queries and keys turn."""
    widths = (heads * d, kv * d, kv * d)
    x, a, b, scale, _ = tables(count, k, widths, r, dtype, seed, t)
    gen = torch.Generator("cuda").manual_seed(seed + 1)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    w, bias = (rand(sum(widths), k) * k ** -0.5).to(dtype), rand(sum(widths))
    positions = torch.randperm(400, generator=torch.Generator().manual_seed(seed))[:t].int().cuda()
    pools = [torch.zeros(t * 2, kv, 4, d, dtype=dtype, device="cuda") for _ in range(2)]
    table = i32([[2 * i + 1] * 100 for i in range(t)])   # (a page for every row's request)
    inv = (1e4 ** (-torch.arange(0, d, 2, dtype=torch.float32) / d)).cuda()
    rows = i32([(i * 5) % (count + 2) - 1 for i in range(t)])   # (none, every one, and a number that names none)
    ranks = [r, max(1, r // 2), 0, r][:count]
    return widths, x, a, b, scale, ranks, rows, w, bias, positions, pools, table, inv


def turned(ops, c, heads, kv, d, adapters, bias=True, write=True):
    widths, x, _, _, _, _, _, w, b, positions, pools, table, inv = c
    qkv, (keys, values) = torch.zeros(x.shape[0], sum(widths), dtype=x.dtype, device="cuda"), [p.clone() for p in pools]
    ops.qkv_rope(x, w, b if bias else None, qkv, positions, torch.arange(x.shape[0], device="cuda").int(), inv, d, heads, kv, d, keys, values,
                 table, 4, write_kv=write, adapters=adapters)
    at = (torch.arange(x.shape[0], device="cuda") * 2 + 1, slice(None), positions.long() % 4)
    return qkv[:, :heads * d], keys[at].reshape(x.shape[0], -1), values[at].reshape(x.shape[0], -1), (keys, values)


@pytest.mark.parametrize("t,k,heads,kv,d,r,count", [(1, 64, 4, 2, 16, 16, 2), (5, 160, 6, 2, 64, 3, 3), (16, 2048, 4, 4, 128, 16, 4), (16, 256, 3, 1, 48, 64, 4),
                                                    (17, 96, 5, 5, 80, 8, 2), (32, 1024, 8, 1, 128, 40, 4)])
@pytest.mark.parametrize("bias", [False, True])
def test_adapters_join_the_sums_of_the_turned_projection(ops, t, k, heads, kv, d, r, count, bias):
    """The one kernel of few bfloat16 rows against the definition in 64 bits: the product's and the adapters' sums in 32 bits, one rounding
    of the turned numbers; rows without an adapter have the bits that they have without any."""
    c = turned_case(t, k, heads, kv, d, r, count, torch.bfloat16, t + k)
    widths, x, a, b, scale, ranks, rows, w, bias_, positions, _, _, inv = c
    assert ops.qkv_rope_takes(x, d, d)
    *got, _ = turned(ops, c, heads, kv, d, (a, b, scale, i32(ranks), widths, rows, 0), bias)
    D, F = torch.float64, 2.0 ** -24
    product, sizes = x.to(D) @ w.to(D).t(), x.to(D).abs() @ w.to(D).abs().t()
    # (32-bit sums: k products, up to 16 parts; the definition's room for 32-bit rows, whose h keeps 24 bits)
    want, room = rc.adapters(x.float(), a.float(), b.float(), scale, ranks, widths, rows, product)
    room = room + (k + 16) * F * sizes + 4 * F * want.abs()
    if bias:
        want, room = want + bias_.to(D), room + 2 * F * (want.abs() + bias_.to(D).abs())
    phi = (positions[:, None].float() * inv[None]).to(D)
    cos, sin = phi.cos()[:, None], phi.sin()[:, None]
    o = 0
    for turns, width, mine in ((True, widths[0], got[0]), (True, widths[1], got[1]), (False, widths[2], got[2])):
        ref, off = want[:, o:o + width].reshape(t, -1, d), room[:, o:o + width].reshape(t, -1, d)
        if turns:   # (sine and cosine of the 32-bit angle within 2^-22)
            (lo, hi), (elo, ehi) = ref.split(d // 2, 2), off.split(d // 2, 2)
            size = lo.abs() + hi.abs()
            ref = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], 2)
            off = torch.cat([elo + ehi + (2.0 ** -22 + 4 * F) * size] * 2, 2)
        rc.close(mine, ref.reshape(t, -1), (off * (1 + 2.0 ** -7) + 2.0 ** -8 * ref.abs()).reshape(t, -1))
        o += width
    *alone, _ = turned(ops, c, heads, kv, d, None, bias)
    none = [i for i, g in enumerate(rows.tolist()) if not 0 <= g < count]
    for g, h in zip(got, alone):
        assert torch.equal(g[none].view(torch.int16), h[none].view(torch.int16))
    q, _, _, pools = turned(ops, c, heads, kv, d, (a, b, scale, i32(ranks), widths, rows, 0), bias, write=False)
    assert torch.equal(q, got[0]) and not any(p.any() for p in pools)


@pytest.mark.parametrize("dtype,t", [(torch.float32, 9), (torch.bfloat16, 33)])
def test_adapters_of_a_turned_projection_in_three_kernels(ops, dtype, t):
    heads, kv, d, k, r, count = 4, 2, 32, 96, 8, 3
    c = turned_case(t, k, heads, kv, d, r, count, dtype, t)
    widths, x, a, b, scale, ranks, rows, w, bias, positions, pools, table, inv = c
    assert not ops.qkv_rope_takes(x, d, d)
    q, keys, values, _ = turned(ops, c, heads, kv, d, (a, b, scale, i32(ranks), widths, rows, min(t, 3)))
    qkv, k2, v2 = torch.zeros(t, sum(widths), dtype=dtype, device="cuda"), pools[0].clone(), pools[1].clone()
    ops.linear(x, w, qkv)
    ops.adapter_add(x, a, b, scale, i32(ranks), widths, rows, qkv)
    ops.rope_kv_write(qkv, bias, positions, torch.arange(t, device="cuda").int(), inv, d, heads, kv, d, k2, v2, table, 4)
    at = (torch.arange(t, device="cuda") * 2 + 1, slice(None), positions.long() % 4)
    assert torch.equal(q, qkv[:, :heads * d]) and torch.equal(keys, k2[at].reshape(t, -1)) and torch.equal(values, v2[at].reshape(t, -1))


def test_adapters_that_do_not_fit_a_turned_projection_are_refused(ops):
    from ninfer_amd.kernels.ops import KernelError
    c = turned_case(4, 64, 4, 2, 16, 8, 2, torch.bfloat16, 3)
    widths, x, a, b, scale, ranks, rows = c[:7]
    for bad in (dict(b=b[:, :-1].contiguous()), dict(b=b[0]), dict(a=a.float()), dict(rows=rows[:3]), dict(scale=scale[:1]), dict(a=a[:, :, :-1].contiguous())):
        g = dict(dict(a=a, b=b, scale=scale, rows=rows), **bad)
        with pytest.raises(KernelError):
            turned(ops, c, 4, 2, 16, (g["a"], g["b"], g["scale"], i32(ranks), widths, g["rows"], 0))
    with pytest.raises(KernelError, match="together"), ops.together():
        turned(ops, c, 4, 2, 16, (a, b, scale, i32(ranks), widths, rows, 0))


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("model", ["A", "B", "C"])
def test_requests_without_an_adapter_keep_their_bits_beside_one_that_has_one(model_dirs, tmp_path, model, graph):
    """bfloat16 steps of few and of more rows, the same tokens with and without an adapter in the last request: the others'
    logits, and the keys and values behind later ones, are the same bits."""
    from ninfer_amd import Chunk
    cfg, _ = util.read_folder(model_dirs[model]["bfloat16"])
    eng = make(model_dirs, model, "bfloat16", use_graph=graph)
    eng.load_adapter("all", adapters_of(tmp_path, cfg, "bfloat16", 0.1)["all"][0])
    toks = [util.random_tokens(60, cfg["vocab_size"], 5 + i) for i in range(4)]
    got = {}
    for name in (None, "all"):
        sessions = [eng.session(name if i == 3 else None) for i in range(4)]
        done, rows = [0] * 4, []
        for cut in ([5, 1, 3, 2], [20, 1, 9, 2], [1, 1, 1, 1], [1, 1, 1, 1], [1, 1, 1, 1], [1, 1, 1, 20], [30, 1, 1, 30], [1, 1, 1, 1]):
            logits = eng.runner.step([Chunk(s.slot, t[d:d + n], [n - 1], s.adapter) for s, t, d, n in zip(sessions, toks, done, cut)])
            done = [d + n for d, n in zip(done, cut)]
            rows.append(logits.float().cpu().numpy())
        got[name] = np.stack(rows)
        for s in sessions:
            s.close()
    assert np.array_equal(got[None][:, :3], got["all"][:, :3])
    assert not np.array_equal(got[None][:, 3], got["all"][:, 3])
    eng.close()
