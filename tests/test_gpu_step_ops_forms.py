"""The decode-step operators around a shared prompt in the forms that test_gpu_step_ops.py does not reach."""
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests import test_gpu_step_ops as base  # noqa: E402
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


# ---- every form of the kernels -------------------------------------------------------------------

FEW, MANY = [(40, 3), (7, 1), (0, 2)], [(29, 500), (3, 211), (1000, 1)]

QKV_FORMS = [
    # D, heads, kv_heads, bs, rot, bias, norms
    # two vectors of a head to a lane: rotated whole, by half
    (32, 7, 3, 8, 32, True, "qk"), (32, 7, 3, 8, 16, False, "qk"),
    (64, 9, 2, 16, 64, True, "qk"), (64, 9, 2, 16, 32, True, "k"),
    (128, 12, 4, 16, 128, True, "qk"), (128, 12, 4, 16, 64, True, "qk"), (128, 5, 5, 48, 64, False, "q"),
    (256, 3, 1, 16, 256, True, "qk"), (256, 3, 1, 16, 128, True, "qk"),
    # vectors by shuffle: 8, 16 and 32 lanes to a head, two vectors to a lane
    (24, 7, 3, 8, 24, True, "qk"), (32, 7, 3, 8, 8, True, "qk"),
    (48, 7, 3, 8, 48, True, "qk"), (64, 9, 2, 16, 16, True, "qk"), (36, 5, 2, 16, 24, False, "k"),
    (96, 7, 3, 16, 96, True, "qk"), (128, 7, 3, 16, 32, True, "q"),
    (192, 3, 2, 16, 96, True, "qk"), (160, 3, 2, 16, 160, True, "qk"), (256, 3, 1, 16, 64, True, "qk"),
    # value by value
    (34, 7, 3, 8, 34, True, "qk"), (66, 7, 3, 16, 20, True, "qk"), (250, 3, 1, 16, 250, True, "q"), (128, 3, 1, 16, 12, True, "qk"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("chunks", [FEW, MANY])
@pytest.mark.parametrize("D,heads,kv_heads,bs,rot,use_bias,norms", QKV_FORMS)
def test_qkv_norm_post_in_every_form(ops, D, heads, kv_heads, bs, rot, use_bias, norms, chunks, in_place):  # noqa: F811
    base.test_qkv_norm_post(ops, D, heads, kv_heads, bs, rot, use_bias, norms, chunks, in_place)


@pytest.mark.parametrize("D,heads,kv_heads,bs,rot,use_bias,norms", QKV_FORMS[:9])
def test_qkv_norm_post_of_more_tokens_than_a_grid_in_every_form(ops, D, heads, kv_heads, bs, rot, use_bias, norms):  # noqa: F811
    # up to 32 CTAs are on an SM: some of them go through two tokens, or with more heads through several
    base.test_qkv_norm_post(ops, D, heads, kv_heads, bs, rot, use_bias, norms, [(29, 5200)], True)


PREFIX_FORMS = [
    # D, heads, kv_heads, bs, groups: blocks that 16 divides and does not divide, up to 8 heads to a KV head and up to 16
    (D, heads, kv_heads, bs, groups)
    for D in (128, 64, 32, 16)
    for heads, kv_heads in ((10, 2), (24, 2))
    for bs in (16, 24, 8)
    for groups in ([(777, [1, 30, 200, None]), (50, []), (129, [2] * 7), (0, [40]), (9, [])],)
]


@pytest.mark.parametrize("D,heads,kv_heads,bs,groups", PREFIX_FORMS)
def test_shared_prefix_attention_in_every_form(ops, D, heads, kv_heads, bs, groups):  # noqa: F811
    c = prefix_case(D + bs, D, heads, kv_heads, bs, groups)
    wide, alone = padded(c), (0, c["max_prefix"] + c["max_suffix"])
    for batch, hints in ((c, None), (c, SHARED), (c, alone), (wide, None), (wide, alone)):
        check_prefix(c, run_prefix(ops, batch, hints), 7.0)


@pytest.mark.parametrize("hints", [None, SHARED, (0, 1000)])
@pytest.mark.parametrize("groups", [[(40, []), (300, [5, 70])], [(300, [5]), (8, []), (8, []), (17, [1, 2])],
                                    [(0, [])] * 40 + [(200, [3, 9])] + [(5, [])] * 40])
def test_shared_prefix_attention_with_groups_of_nobody(ops, groups, hints):  # noqa: F811
    c = prefix_case(33, 64, 8, 2, 16, groups)
    check_prefix(c, run_prefix(ops, c, hints), 7.0)


def test_refusals_of_device_tensors_launch_nothing(ops):  # noqa: F811
    from relay_b200 import _lib
    f32, f16, i32 = (dict(dtype=t, device="cuda") for t in (torch.float32, torch.float16, torch.int32))
    T, H, KV, D, bs, V = 3, 4, 2, 64, 16, 100
    width = (H + 2 * KV) * D
    meta = ops.TokenMeta(*(torch.zeros(n, **i32) for n in (T, T, 1, 1)))
    short = ops.TokenMeta(meta.pos[:2], meta.seq, meta.table_off, meta.tables)
    host = ops.TokenMeta(meta.pos.cpu(), meta.seq, meta.table_off, meta.tables)
    pool = torch.zeros(2, KV, bs, D, **f16)
    qkv, q, out, inv, norm = torch.zeros(T, width, **f32), torch.zeros(T, H * D, **f32), torch.zeros(T, H * D, **f16), torch.zeros(32, **f32), torch.ones(D, **f32)

    def norm_post(**kw):
        a = dict(qkv=qkv, bias=None, q_norm=norm, k_norm=norm, eps=1e-6, inv_freq=inv, meta=meta, q_out=q, k_pool=pool, v_pool=pool,
                 heads=H, kv_heads=KV, head_dim=D, block_size=bs, rot_dim=None)
        ops.qkv_norm_post(**(a | kw))

    def prefix(**kw):
        a = dict(shape=ops.attn_shape(H, KV, D, bs, q_stride=H * D), q=q, meta=meta, decode_tokens=torch.arange(T, **i32),
                 group_off=torch.tensor([0, T], **i32), prefix_len=torch.zeros(1, **i32), max_prefix=0, max_suffix=1, k_pool=pool, v_pool=pool,
                 out=out, scratch=None)
        ops.shared_prefix_attention(**(a | kw))

    logits = torch.zeros(T, V, **f32)
    ids, lens = torch.zeros(T, 5, **i32), torch.zeros(T, **i32)

    def adjust(**kw):
        a = dict(logits=logits, out=logits, penalties=torch.ones(T, 4, **f32), history=ids, history_len=lens, prompt_len=lens, bias_ids=ids,
                 bias_values=torch.zeros(T, 5, **f32), bias_len=lens, mask=torch.zeros(T, 4, **i32))
        ops.adjust_logits(**(a | kw))

    refused = [
        (norm_post, dict(qkv=qkv.half()), "float32"), (norm_post, dict(qkv=qkv[:, 1:]), "head_dim"), (norm_post, dict(qkv=qkv.t().contiguous().t()), "contiguous"),
        (norm_post, dict(q_out=q[:2]), "q_out"), (norm_post, dict(meta=short), "metadata"), (norm_post, dict(meta=host), "device"),
        (norm_post, dict(k_pool=pool[:, :1].contiguous()), "pools"), (norm_post, dict(v_pool=pool[:1]), "pools"), (norm_post, dict(v_pool=pool.transpose(1, 2)), "contiguous"),
        (norm_post, dict(bias=norm), "bias"), (norm_post, dict(k_norm=inv), "q_norm and k_norm"), (norm_post, dict(rot_dim=32), "inv_freq"),
        (norm_post, dict(rot_dim=66, inv_freq=torch.zeros(33, **f32)), "rot_dim"),
        (prefix, dict(q=q[:2]), "rows"), (prefix, dict(out=out[:2]), "rows"), (prefix, dict(out=out.float()), "float16"), (prefix, dict(q=qkv), "apart"),
        (prefix, dict(group_off=torch.zeros(3, **i32)), "group_off"), (prefix, dict(decode_tokens=torch.arange(T, device="cuda")), "int32"),
        (prefix, dict(k_pool=pool[:, :, :8].contiguous()), "pools"), (prefix, dict(scratch=torch.zeros(8, **f32)), "uint8"), (prefix, dict(max_prefix=-1), "bad batch"),
        (prefix, dict(max_prefix=100000, scratch=torch.zeros(16, dtype=torch.uint8, device="cuda")), "scratch too small"),
        (adjust, dict(out=torch.zeros(T, V + 1, **f32)), "vocabulary"), (adjust, dict(out=torch.zeros(1, V, **f32).expand(T, V)), "shorter"),
        (adjust, dict(penalties=torch.ones(T, 3, **f32)), "penalties"), (adjust, dict(history=None), "history"), (adjust, dict(history_len=lens[:2]), "history"),
        (adjust, dict(history=ids.long()), "int32"), (adjust, dict(bias_values=None), "bias_ids"), (adjust, dict(bias_len=lens[:1]), "bias_ids"),
        (adjust, dict(mask=torch.zeros(T, 3, **i32)), "mask"), (adjust, dict(mask=torch.zeros(1, 4, **i32)), "mask"),
    ]
    before = _lib.lib().rb200_kernel_launches()
    for call, kw, text in refused:
        with pytest.raises(ValueError, match=text):
            call(**kw)
    assert _lib.lib().rb200_kernel_launches() == before
    for call in (norm_post, prefix, adjust):
        call()
    torch.cuda.synchronize()
    assert _lib.lib().rb200_kernel_launches() == before + 3


FIRST_CALLS_FROM_SEVERAL_THREADS = """
import threading
import torch
from relay_b200 import ops
i32 = dict(dtype=torch.int32, device="cuda")
shape = ops.attn_shape(8, 2, 128, 16)
pool = torch.randn(40, 2, 16, 128, device="cuda").half()
q = torch.randn(1, 12 * 128, device="cuda")
meta = ops.TokenMeta(torch.tensor([599], **i32), torch.tensor([0], **i32), torch.tensor([0], **i32), torch.arange(40, **i32))
args = shape, q, meta, torch.tensor([0], **i32), torch.tensor([0, 1], **i32), torch.tensor([590], **i32)
logits = torch.randn(300, 60000, device="cuda")
torch.cuda.synchronize()
ready, results = threading.Barrier(8), [None] * 8

def work(n):
    with torch.cuda.stream(torch.cuda.Stream()):
        out, adjusted = torch.zeros(1, 1024, dtype=torch.float16, device="cuda"), torch.empty_like(logits)
        ready.wait()
        ops.shared_prefix_attention(*args, 1 << 20, 0, pool, pool, out)
        ops.adjust_logits(logits, adjusted)
        torch.cuda.current_stream().synchronize()
        results[n] = out, adjusted

threads = [threading.Thread(target=work, args=(n,)) for n in range(8)]
for t in threads: t.start()
for t in threads: t.join()
assert all(r is not None and torch.equal(r[0], results[0][0]) and torch.equal(r[1], logits) for r in results)
assert results[0][0].abs().max() > 0
"""


def test_first_calls_of_several_threads_at_once():
    # in a process of its own, whose kernels' shared-memory limits nobody has raised yet
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS_FROM_SEVERAL_THREADS], timeout=300, cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
