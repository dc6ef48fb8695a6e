"""The decode-step operators around a shared prompt in the forms that test_gpu_step_ops.py does not reach."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_gpu_step_ops import (H16, NORM_TOL, SHARED, U32, check_prefix, dev, norm_rope_f64, ops,  # noqa: E402, F401
                                     padded, prefix_case, run_prefix)


@pytest.mark.parametrize("T", [1, 2, 5])
def test_qkv_norm_post_in_place_through_a_view_of_the_query_part(ops, T):  # noqa: F811
    # torch counts a single row as contiguous, whatever the view's stride
    rng = np.random.Generator(np.random.PCG64(T))
    heads, kv_heads, D, bs = 6, 2, 64, 16
    x = rng.standard_normal((T, (heads + 2 * kv_heads) * D)).astype(np.float32)
    qn, kn = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    inv = (10000.0 ** -(np.arange(0, D, 2) / D)).astype(np.float32)
    pos = np.arange(T) + 9
    meta = ops.TokenMeta.from_host(pos, np.zeros(T), [0], [0])
    pools = [torch.zeros((1, kv_heads, bs, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    qkv = dev(x)
    got = ops.qkv_norm_post(qkv, None, dev(qn), dev(kn), 1e-6, dev(inv), meta, qkv[:, :heads * D], *pools, heads, kv_heads, D, bs)
    q, _, v, reach = norm_rope_f64(x, None, qn, kn, 1e-6, inv, pos, heads, kv_heads, D, D)
    assert got.data_ptr() == qkv.data_ptr()
    after = qkv.cpu().numpy()
    assert np.all(np.abs(after[:, :heads * D].reshape(q.shape) - q) <= NORM_TOL * reach[:, :heads])
    assert np.array_equal(after[:, heads * D:], x[:, heads * D:])
    assert np.array_equal(pools[1].cpu().numpy()[0, :, 9:9 + T].transpose(1, 0, 2), v.astype(np.float16))


def check_penalised(got, x, rep):
    """`got` against x / rep for x > 0 and x rep for the others, in float64."""
    wide, rep = x.astype(np.float64), rep.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        want = np.where(wide > 0, wide / rep, wide * rep)
        nearest = want.astype(np.float32)
    finite = np.isfinite(nearest)
    assert np.array_equal(got[~finite], nearest[~finite], equal_nan=True)
    # Half a step of float32 (2^-22 of one more for a quotient), or of its subnormals. Quotients outside of 2^-99 to 2^100
    # are products with a reciprocal: each of the two rounds, and where the type's range ends below so does the
    # scaled logit (half a subnormal step, times a reciprocal of at most 2).
    size = np.abs(want[finite])
    twice = (wide[finite] > 0) & ((size <= 2.0 ** -99) | (size >= 2.0 ** 100))
    tol = np.where(twice, 2 * U32 * size + 3 * 2.0 ** -150, U32 * (1 + 2.0 ** -22) * size + 2.0 ** -150)
    assert np.all(np.abs(got[finite] - want[finite]) <= tol)


@pytest.mark.parametrize("repetition", [1e-39, 2.0 ** -128, 0.7, 1.1, 3.0, 1e38])
def test_adjust_logits_divides_by_the_repetition(ops, repetition):  # noqa: F811
    # also where 1 / repetition is no float32
    R, V = 3, 5000
    x = np.random.Generator(np.random.PCG64(2)).standard_normal((R, V)).astype(np.float32)
    x *= np.float32(1e-3 if repetition < 1 else 4)
    pen = np.zeros((R, 4), np.float32)
    pen[:, 0] = repetition
    history = np.broadcast_to(np.arange(V, dtype=np.int32), (R, V))
    out = torch.empty((R, V), device="cuda")
    ops.adjust_logits(dev(x), out, dev(pen), dev(history), dev(np.full(R, V, np.int32)))
    check_penalised(out.cpu().numpy(), x, pen[:, :1])


def test_adjust_logits_divides_by_the_repetition_at_every_magnitude(ops):  # noqa: F811
    rng = np.random.Generator(np.random.PCG64(7))
    R, V = 120, 3001
    x = (rng.standard_normal((R, V)) * 2.0 ** rng.integers(-140, 120, (R, V))).astype(np.float32)
    x[:, 0], x[:, 1], x[:, 2] = np.inf, -np.inf, np.nan
    pen = np.zeros((R, 4), np.float32)
    pen[:, 0] = (1 + rng.random(R)) * 2.0 ** rng.integers(-30, 30, R)
    history = np.broadcast_to(np.arange(V, dtype=np.int32), (R, V))
    out = torch.empty((R, V), device="cuda")
    ops.adjust_logits(dev(x), out, dev(pen), dev(history), dev(np.full(R, V, np.int32)))
    check_penalised(out.cpu().numpy(), x, pen[:, :1])


@pytest.mark.parametrize("D,bs", [(128, 1 << 23), (80, 1 << 24), (66, 1 << 24)])
def test_qkv_norm_post_into_a_block_of_more_than_2_31_values(ops, D, bs):  # noqa: F811
    # one block per sequence, as long as its context may get: the third KV head begins 2^31 values in or later
    heads, kv_heads, T = 2, 3, 3
    rng = np.random.Generator(np.random.PCG64(D))
    x = rng.standard_normal((T, (heads + 2 * kv_heads) * D)).astype(np.float32)
    pos = np.asarray([0, bs - 2, bs - 1])
    inv = (500000.0 ** -(np.arange(0, D, 2) / D)).astype(np.float32)
    pools = [torch.zeros((1, kv_heads, bs, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    q_out = torch.empty((T, heads * D), device="cuda")
    ops.qkv_norm_post(dev(x), None, None, None, 1e-6, dev(inv), ops.TokenMeta.from_host(pos, np.zeros(T), [0], [0]), q_out, *pools,
                      heads, kv_heads, D, bs)
    q, k, v, reach = norm_rope_f64(x, None, None, None, 1e-6, inv, pos, heads, kv_heads, D, D)
    assert np.all(np.abs(q_out.cpu().numpy().reshape(q.shape) - q) <= NORM_TOL * reach[:, :heads])
    got = [pool[0][:, torch.from_numpy(pos).cuda()].cpu().numpy().transpose(1, 0, 2) for pool in pools]
    tol = H16 * np.abs(k) + 2.0 ** -25 + NORM_TOL * reach[:, heads:heads + kv_heads]
    assert np.all(np.abs(got[0].astype(np.float64) - k) <= tol)
    assert np.array_equal(got[1], v.astype(np.float16))
    for pool, here in zip(pools, got):  # nothing went anywhere else
        assert sum(int(torch.count_nonzero(pool[0, h])) for h in range(kv_heads)) == np.count_nonzero(here)


@pytest.mark.parametrize("D,bs", [(128, 16), (64, 24), (64, 8), (32, 8), (16, 1)])
def test_shared_prefix_attention_follows_tables_rewritten_in_place(ops, D, bs):  # noqa: F811
    # a captured step whose block tables, pages and queries change between replays, in kernels and copies just ahead of it
    c = prefix_case(31, D, 8, 2, bs, [(900, [1, 40, 333]), (70, [5, 200])])
    shape = ops.attn_shape(8, 2, D, bs, o_stride=c["o_stride"])
    meta = ops.TokenMeta.from_host(c["pos"], c["seq"], c["table_off"], c["tables"])
    pools = [dev(np.nan_to_num(c[name])) for name in ("k", "v")]
    tables, pages, queries = meta.tables.clone(), [p.clone() for p in pools], dev(c["q"])
    q, out = queries.clone(), torch.full((len(c["pos"]), c["o_stride"]), 7.0, dtype=torch.float16, device="cuda")
    scratch = torch.empty(ops.shared_prefix_scratch_bytes(shape, 5, 2, *SHARED), dtype=torch.uint8, device="cuda")
    args = dev(c["tokens"]), dev(c["off"]), dev(c["lens"]), *SHARED, *pools, out, scratch
    nb = len(c["k"])
    order = torch.arange(nb, device="cuda")

    def step():
        # the same batch with its blocks elsewhere in the pool
        meta.tables.copy_(order[tables.long()].int())
        for pool, page in zip(pools, pages):
            pool[order] = page
        q.copy_(queries)
        ops.shared_prefix_attention(shape, q, meta, *args)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for shift in range(8):
        order.copy_((torch.arange(nb, device="cuda") + 3 * shift) % nb)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check_prefix(c, out.cpu().numpy(), 7.0)


# ---- queries that fp16 does not hold -------------------------------------------------------------

HOT = 60.0  # score of two keys of each context; all others score 0


def competing_case(seed, D, heads, kv_heads, bs, groups, where):
    """A prefix_case in which two keys of each context share the weight, their scores nearly equal and so large that
    rounding the query to fp16 would move the weights visibly. `where`: 's' and 'o' for shared and own keys."""
    c = prefix_case(seed, D, heads, kv_heads, bs, groups, dtype_q=np.float32)
    rng = np.random.Generator(np.random.PCG64(seed))
    n = len(c["q"])
    c["q"][:, :heads * D] = 30 * (1 + 2.0 ** -9 * rng.uniform(-1, 1, (n, heads * D)))  # some seven steps of fp16 wide
    c["k"][~np.isnan(c["k"])] = 0
    hot = np.float16(HOT * np.sqrt(D) / 30)
    i = 0
    for P, own in groups:
        shared = rng.permutation(P)[:2]
        for s in own:
            ctx, tok = c["contexts"][i], c["tokens"][i]
            ctx[0] = 0
            mine = P + rng.permutation(s)[:2]
            for j, (kind, dim) in enumerate(zip(where, (3, D - 2))):  # each of the two keys looks at one dimension
                key = shared[j] if kind == "s" else mine[j]
                page = c["tables"][c["table_off"][c["seq"][tok]] + key // bs]
                ctx[0, key, :, dim] = c["k"][page, :, key % bs, dim] = hot
            i += 1
    return c


def check_unrounded(c, out):
    """Each decode token against float64, with nothing granted for a rounding of q; and what such a rounding would do."""
    D, G = c["D"], c["heads"] // c["kv_heads"]

    def attend(q, ctx):
        k, v = (ctx[i].astype(np.float64).transpose(1, 0, 2) for i in (0, 1))
        s = q.reshape(c["kv_heads"], G, D) @ k.transpose(0, 2, 1) / np.sqrt(D)
        w = np.exp(s - s.max(-1, keepdims=True))
        total = w.sum(-1, keepdims=True)
        return w / total @ v, w / total @ np.abs(v), total

    for tok, ctx in zip(c["tokens"], c["contexts"]):
        q = c["q"][tok, :c["heads"] * D]
        want, spread, total = attend(q.astype(np.float64), ctx)
        # Weights and output round to fp16 (2^-11 each; weights below 2^-14 of the largest to 2^-25). Scores are single
        # products: q = hi + lo to 2^-22, three roundings to float32, 60 (2^-22 + 3 2^-24) = 2.5e-5 < 2^-15; such an
        # error of both scores moves the output by 2^-15 of the spread at most, as do exponentials and sums.
        tol = (H16 + 2 * 2.0 ** -15) * spread + H16 * np.abs(want) + ctx.shape[1] * 2.0 ** -25 * np.abs(ctx[1]).max() / total + 2.0 ** -25
        rounded, _, _ = attend(q.astype(np.float16).astype(np.float64), ctx)
        assert (np.abs(rounded - want) / tol).max() > 4, "the case would not notice a query rounded to fp16"
        if out is not None:
            got = out[tok, :c["heads"] * D].astype(np.float64).reshape(want.shape)
            assert (np.abs(got - want) / tol).max() <= 1, (tok, (np.abs(got - want) / tol).max())


COMPETING = [
    # D, heads, kv_heads, bs, groups
    (128, 32, 8, 16, [(700, [5, 40]), (130, [2, 17, 300])]),
    (128, 32, 8, 16, [(700, [2 + i for i in range(40)])]),   # more than 64 rows to a group
    (64, 10, 2, 16, [(700, [5, 40]), (130, [2, 17, 300])]),
    (64, 10, 2, 16, [(700, [2 + i for i in range(40)])]),
    (128, 8, 2, 8, [(500, [5, 40, 130])]),
    (64, 32, 2, 24, [(500, [5, 40, 130])]),
    (32, 8, 2, 8, [(500, [5, 40, 130])]),
    (32, 32, 2, 16, [(500, [5, 40, 130])]),
    (16, 16, 1, 8, [(500, [5, 40, 130])]),
]


@pytest.mark.parametrize("where", ["ss", "oo", "so"])
@pytest.mark.parametrize("D,heads,kv_heads,bs,groups", COMPETING)
def test_shared_prefix_attention_takes_queries_in_full(ops, D, heads, kv_heads, bs, groups, where):  # noqa: F811
    c = competing_case(D + heads, D, heads, kv_heads, bs, groups, where)
    check_unrounded(c, run_prefix(ops, c))
    check_unrounded(c, run_prefix(ops, c, SHARED))
    check_unrounded(c, run_prefix(ops, c, (0, c["max_prefix"] + c["max_suffix"])))
    wide = padded(c)
    check_unrounded(c, run_prefix(ops, wide))
    check_unrounded(c, run_prefix(ops, wide, (0, c["max_prefix"] + c["max_suffix"])))
