"""The decode-step operators around a shared prompt (qkv_norm_post, shared_prefix_attention,
adjust_logits) against their definitions in float64, at the sizes, masks and layouts where they can
go wrong, and a run of them together as a step uses them."""
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from oracle import oracle  # noqa: E402

H16, U32 = 2.0 ** -11, 2.0 ** -24  # half a step of fp16 and of float32, relative


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from relay_b200 import ops as o
    return o


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- norms, rotation, append ------------------------------------------------------------------


def norm_rope_f64(qkv, bias, q_norm, k_norm, eps, inv_freq, pos, heads, kv_heads, D, rot):
    """(q, k, v, reach): float64 results and, per q and k value, the magnitude its rounding errors refer to."""
    x = qkv.astype(np.float64) + (0 if bias is None else bias.astype(np.float64))
    x = x.reshape(len(x), heads + 2 * kv_heads, D)
    y = x.copy()
    for part, w in ((slice(0, heads), q_norm), (slice(heads, heads + kv_heads), k_norm)):
        if w is not None:
            y[:, part] = x[:, part] / np.sqrt((x[:, part] ** 2).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    angle = pos.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
    h = rot // 2
    a, b = y[:, :heads + kv_heads, :h].copy(), y[:, :heads + kv_heads, h:rot].copy()
    reach = np.abs(y)
    reach[:, :heads + kv_heads, :h] = reach[:, :heads + kv_heads, h:rot] = np.abs(a) + np.abs(b)
    y[:, :heads + kv_heads, :h] = a * np.cos(angle) - b * np.sin(angle)
    y[:, :heads + kv_heads, h:rot] = b * np.cos(angle) + a * np.sin(angle)
    return y[:, :heads], y[:, heads:heads + kv_heads], y[:, heads + kv_heads:], reach


# Half steps of float32 in q: the sum of squares at most D/32 + 5 = 13, mean, eps, root, quotient and
# the two products 6, the two terms of the rotation 3, the angle (at most pi, rounded once: 2 pi) and
# sincosf's own 2 units in the last place 4: 33 of the pair's magnitude.
NORM_TOL = 33 * U32

QKV_CASES = [
    # D, heads, kv_heads, bs, rot, bias, norms, chunks (start, tokens)
    (128, 32, 8, 16, 128, False, "qk", [(4000, 1), (131071, 1), (0, 1)]),
    (128, 32, 8, 16, 128, True, "qk", [(5, 19), (16, 16), (0, 33)]),
    (64, 16, 16, 32, 32, True, "qk", [(31, 2), (77, 1)]),
    (64, 14, 2, 64, 64, False, "k", [(1000, 70)]),
    (80, 9, 3, 8, 80, False, "qk", [(3, 9), (100, 1)]),
    (80, 9, 3, 8, 40, True, "q", [(3, 9)]),
    (256, 8, 1, 16, 256, False, "qk", [(15, 3), (2000, 1)]),
    (256, 8, 4, 16, 64, True, "qk", [(15, 3)]),
    (16, 4, 2, 16, 16, True, "qk", [(0, 5)]),
    (8, 8, 2, 32, 8, False, "qk", [(40, 5)]),
    (2, 3, 3, 1, 2, False, "qk", [(0, 4)]),
    (128, 4, 4, 48, 0, False, "qk", [(40, 20)]),
    (128, 16, 1, 16, 128, True, "", [(40, 20)]),
    (120, 6, 2, 16, 60, True, "qk", [(9, 8)]),
    (96, 40, 8, 16, 96, False, "qk", [(1 << 20, 5)]),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("D,heads,kv_heads,bs,rot,use_bias,norms,chunks", QKV_CASES)
def test_qkv_norm_post(ops, D, heads, kv_heads, bs, rot, use_bias, norms, chunks, in_place):
    rng = np.random.Generator(np.random.PCG64(D + heads))
    width, pad = (heads + 2 * kv_heads) * D, 0 if in_place else 12
    pos, seq, off, tables, used = [], [], [], [], 0
    for s, (start, n) in enumerate(chunks):
        first, last = start // bs, (start + n - 1) // bs
        off.append(len(tables))
        tables += [0] * first + [(3 + used + i) for i in range(last - first + 1)]
        used += last - first + 1
        pos += range(start, start + n)
        seq += [s] * n
    nb = used + 5
    T = len(pos) + 2  # two padding tokens behind the last sequence
    pos, seq = np.asarray(pos + [7, -1], np.int32), np.asarray(seq + [-1, 0], np.int32)
    off, tables = np.asarray(off, np.int32), np.asarray(tables, np.int32)
    qkv = np.full((T, width + pad), np.nan, np.float32)
    qkv[:, :width] = rng.standard_normal((T, width)) * 2
    qkv[-2:] = np.nan  # padding: neither read nor written
    bias = (0.1 * rng.standard_normal(width)).astype(np.float32) if use_bias else None
    qn = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32) if "q" in norms else None
    kn = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32) if "k" in norms else None
    inv = (500000.0 ** -(np.arange(0, max(rot, 2), 2) / max(rot, 2))).astype(np.float32)[:rot // 2]
    g_qkv = dev(qkv)
    q_out = g_qkv if in_place else torch.full((T, heads * D + 4), 5.0, device="cuda")
    kp = torch.full((nb, kv_heads, bs, D), 9.0, dtype=torch.float16, device="cuda")
    vp = kp.clone()
    meta = ops.TokenMeta.from_host(pos, seq, off, tables)
    opt = lambda a: None if a is None else dev(a)  # noqa: E731
    ops.qkv_norm_post(g_qkv, opt(bias), opt(qn), opt(kn), 1e-6, dev(inv), meta, q_out, kp, vp, heads, kv_heads, D, bs, rot_dim=rot)
    n = T - 2
    q, k, v, reach = norm_rope_f64(qkv[:n, :width], bias, qn, kn, 1e-6, inv, pos[:n], heads, kv_heads, D, rot)
    got = q_out.cpu().numpy()
    assert np.all(np.abs(got[:n, :heads * D].reshape(q.shape) - q) <= NORM_TOL * reach[:, :heads] + 1e-30)
    after = g_qkv.cpu().numpy()
    if in_place:
        assert np.array_equal(after[:n, heads * D:], qkv[:n, heads * D:], equal_nan=True)
        assert np.all(np.isnan(after[n:]))
    else:
        assert np.array_equal(after, qkv, equal_nan=True)
        assert np.all(got[:n, heads * D:] == 5) and np.all(got[n:] == 5)
    want_v = (qkv[:n, :width] + (0 if bias is None else bias)).astype(np.float32).reshape(n, -1, D)[:, heads + kv_heads:].astype(np.float16)
    written = np.zeros((nb, bs), bool)
    gk, gv = kp.cpu().numpy(), vp.cpu().numpy()
    for t in range(n):
        page, slot = tables[off[seq[t]] + pos[t] // bs], pos[t] % bs
        written[page, slot] = True
        tol = H16 * np.abs(k[t]) + 2.0 ** -25 + NORM_TOL * reach[t, heads:heads + kv_heads]
        assert np.all(np.abs(gk[page, :, slot].astype(np.float64) - k[t]) <= tol)
        assert np.array_equal(gv[page, :, slot], want_v[t])
    rest = np.broadcast_to(~written[:, None, :, None], gk.shape)
    assert np.all(gk[rest] == 9) and np.all(gv[rest] == 9)  # no other slot is touched


@pytest.mark.parametrize("D,rot", [(128, 128), (64, 32), (80, 80)])
@pytest.mark.parametrize("shift,pad", [(1, 3), (2, 0), (0, 1)])
def test_qkv_norm_post_of_unaligned_rows(ops, D, rot, shift, pad):
    # rows that start anywhere in memory: the same values as from aligned ones, up to the order of a head's sum
    rng = np.random.Generator(np.random.PCG64(D + shift))
    heads, kv_heads, bs, T = 6, 2, 16, 21
    width = (heads + 2 * kv_heads) * D
    flat = torch.zeros(shift + T * (width + pad), device="cuda")
    qkv = flat[shift:].view(T, width + pad)
    qkv[:, :width] = dev(rng.standard_normal((T, width)).astype(np.float32))
    qn, kn = (dev((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2))
    inv = (10000.0 ** -(np.arange(0, rot, 2) / rot)).astype(np.float32)
    meta = ops.TokenMeta.from_host(np.arange(T) + 5, np.zeros(T), [0], [1, 0])
    kp = torch.zeros((2, kv_heads, bs, D), dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    q_out = torch.zeros((T, heads * D + 1), device="cuda")
    ops.qkv_norm_post(qkv, None, qn, kn, 1e-6, dev(inv), meta, q_out, kp, vp, heads, kv_heads, D, bs, rot_dim=rot)
    q, k, v, reach = norm_rope_f64(qkv[:, :width].cpu().numpy(), None, qn.cpu().numpy(), kn.cpu().numpy(), 1e-6, inv,
                                   np.arange(T) + 5, heads, kv_heads, D, rot)
    got = q_out.cpu().numpy()
    assert np.all(np.abs(got[:, :heads * D].reshape(q.shape) - q) <= NORM_TOL * reach[:, :heads])
    assert np.all(got[:, heads * D:] == 0)
    gv = vp.cpu().numpy()
    for t in range(T):
        assert np.array_equal(gv[[1, 0][(t + 5) // bs], :, (t + 5) % bs], v[t].astype(np.float16))


def test_qkv_norm_post_of_more_tokens_than_the_grid_holds(ops):
    # many tokens, padding among them: a CTA goes through several
    rng = np.random.Generator(np.random.PCG64(11))
    heads, kv_heads, D, bs, T = 4, 1, 64, 16, 6001
    width = (heads + 2 * kv_heads) * D
    qkv = rng.standard_normal((T, width)).astype(np.float32)
    pos, seq = np.arange(T, dtype=np.int32), np.zeros(T, np.int32)
    pad = rng.random(T) < 0.1
    pad[[0, T - 1]] = True
    seq[pad] = -1
    inv = (10000.0 ** -(np.arange(0, D, 2) / D)).astype(np.float32)
    nb = (T + bs - 1) // bs
    table = rng.permutation(nb).astype(np.int32)
    meta = ops.TokenMeta.from_host(pos, seq, [0], table)
    kp = torch.full((nb, kv_heads, bs, D), 9.0, dtype=torch.float16, device="cuda")
    vp = kp.clone()
    q_out = torch.full((T, heads * D), 5.0, device="cuda")
    ops.qkv_norm_post(dev(qkv), None, None, None, 1e-6, dev(inv), meta, q_out, kp, vp, heads, kv_heads, D, bs)
    q, k, v, reach = norm_rope_f64(qkv, None, None, None, 1e-6, inv, pos, heads, kv_heads, D, D)
    got = q_out.cpu().numpy().reshape(q.shape)
    assert np.all(got[pad] == 5) and np.all(np.abs(got - q)[~pad] <= NORM_TOL * reach[:, :heads][~pad])
    rows = vp[torch.from_numpy(table).long()].transpose(1, 2).reshape(nb * bs, kv_heads, D)[:T].cpu().numpy()
    assert np.all(rows[pad] == 9) and np.array_equal(rows[~pad], v[~pad].astype(np.float16))


def test_qkv_norm_post_without_norms_agrees_with_qkv_post(ops):
    rng = np.random.Generator(np.random.PCG64(5))
    heads, kv_heads, D, bs, T = 8, 2, 64, 16, 40
    qkv = rng.standard_normal((T, (heads + 2 * kv_heads) * D)).astype(np.float32)
    inv = (10000.0 ** -(np.arange(0, D, 2) / D)).astype(np.float32)
    meta = ops.TokenMeta.from_host(np.arange(T), np.zeros(T), [0], [2, 0, 1])
    pools = [torch.zeros((3, kv_heads, bs, D), dtype=torch.float16, device="cuda") for _ in range(4)]
    a, b = dev(qkv), dev(qkv)
    ops.qkv_post(a, None, dev(inv), meta, pools[0], pools[1], heads, kv_heads, D, bs)
    ops.qkv_norm_post(b, None, None, None, 1e-6, dev(inv), meta, b, pools[2], pools[3], heads, kv_heads, D, bs)
    # positions below 40: the float32 product of the angle there is off by at most 40 * 2^-24
    assert (a[:, :heads * D] - b[:, :heads * D]).abs().max().item() <= (40 + 20) * U32 * 2 * np.abs(qkv).max()
    assert torch.equal(pools[1], pools[3])


# ---- attention over a shared prefix ------------------------------------------------------------


def prefix_case(seed, D, heads, kv_heads, bs, groups, peaked=1.0, q_pad=0, o_pad=0, dtype_q=np.float16):
    """A batch of decode tokens in groups: [(shared keys, [own keys of each member, or None for padding])].
    A member is described by its own keys behind the prefix; a negative number takes that many keys off
    the prefix (a context that ends inside it). Batch rows are shuffled; unused slots of the pool hold NaN."""
    rng = np.random.Generator(np.random.PCG64(seed))
    members = [(g, P, s) for g, (P, own) in enumerate(groups) for s in own]
    n = len(members)
    rows = rng.permutation(n + 3)[:n]  # three batch rows are no decode tokens
    pos, seq = np.full(n + 3, -5, np.int32), np.full(n + 3, -1, np.int32)
    sizes = [len(own) for _, own in groups]
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    lens = np.asarray([P for P, _ in groups], np.int32)
    tokens, tables, table_off, contexts, need = [], [], [], [], 0
    shared = {}
    for g, (P, own) in enumerate(groups):
        kv = rng.standard_normal((2, P, kv_heads, D)).astype(np.float16)
        shared[g] = (kv, list(range(need, need + P // bs)))
        need += P // bs
    fills = []  # (block, slots, k, v)
    for i, (g, P, s) in enumerate(members):
        if s is None:
            tokens.append(-1)
            contexts.append(None)
            continue
        ctx = P + s
        kv, whole = shared[g]
        own_kv = rng.standard_normal((2, max(s, 0), kv_heads, D)).astype(np.float16)
        full = np.concatenate([kv[:, :min(P, ctx)], own_kv], 1)
        blocks = whole[:min(P, ctx) // bs]
        while len(blocks) * bs < ctx:
            blocks = blocks + [need]
            need += 1
        for b in range((ctx + bs - 1) // bs):
            part = full[:, b * bs:(b + 1) * bs]
            if b >= len(whole) or b * bs + bs > min(P, ctx):
                fills.append((blocks[b], part))
        tables += [0] * (i % 3)  # tables start anywhere
        table_off.append(len(tables))
        tables += blocks
        tokens.append(rows[i])
        pos[rows[i]], seq[rows[i]] = ctx - 1, len(table_off) - 1
        contexts.append(full)
    for g, (kv, whole) in shared.items():
        for b, block in enumerate(whole):
            fills.append((block, kv[:, b * bs:(b + 1) * bs]))
    nb = need + 2
    perm = rng.permutation(nb).astype(np.int32)
    pools = np.full((2, nb, kv_heads, bs, D), np.nan, np.float16)
    for block, part in fills:
        pools[:, perm[block], :, :part.shape[1]] = part.transpose(0, 2, 1, 3)
    q = np.full((n + 3, (heads + 2 * kv_heads) * D + q_pad), np.nan, np.float32)
    q[:, :heads * D] = (rng.standard_normal((n + 3, heads * D)) * peaked).astype(dtype_q)
    return dict(D=D, heads=heads, kv_heads=kv_heads, bs=bs, pos=pos, seq=seq, table_off=np.asarray(table_off or [0], np.int32),
                tables=perm[np.asarray(tables or [0])], tokens=np.asarray(tokens, np.int32), off=off, lens=lens, q=q, k=pools[0],
                v=pools[1], contexts=contexts, o_stride=heads * D + o_pad, max_prefix=int(lens.max(initial=0)),
                max_suffix=max([s for _, _, s in members if s is not None], default=0))


def check_prefix(c, out, untouched):
    """Each decode token's row against softmax(q K^T / sqrt D) V in float64."""
    D, G = c["D"], c["heads"] // c["kv_heads"]
    seen = np.zeros(len(out), bool)
    for tok, ctx in zip(c["tokens"], c["contexts"]):
        if tok < 0:
            continue
        seen[tok] = True
        got = out[tok, :c["heads"] * D].astype(np.float64).reshape(c["kv_heads"], G, D)
        if ctx.shape[1] == 0:
            assert np.all(got == 0)
            continue
        q = c["q"][tok, :c["heads"] * D].astype(np.float64).reshape(c["kv_heads"], G, D)
        k, v = (ctx[i].astype(np.float64).transpose(1, 0, 2) for i in (0, 1))  # [kv_heads, keys, D]
        s = q @ k.transpose(0, 2, 1) / np.sqrt(D)
        w = np.exp(s - s.max(-1, keepdims=True))
        total = w.sum(-1, keepdims=True)
        w /= total
        want, spread = w @ v, w @ np.abs(v)
        # q rounds to fp16: a score moves by up to 2^-11 sum |q k| / sqrt D, the output by that times |v - o|
        q16 = q.astype(np.float16).astype(np.float64)
        moved = (np.abs(q - q16) @ np.abs(k).transpose(0, 2, 1)) / np.sqrt(D)
        q_err = (w * moved) @ np.abs(v) + (w * moved).sum(-1, keepdims=True) * np.abs(want)
        # each weight rounds to fp16 (2^-11 of it, or 2^-25 of the largest where it is subnormal), so does
        # the output; scores, exponentials and sums in float32 stay within 2^-15
        tol = (H16 + 2.0 ** -15) * spread + H16 * np.abs(want) + 1.05 * q_err + ctx.shape[1] * 2.0 ** -25 * np.abs(v).max() / total + 2.0 ** -25
        worst = (np.abs(got - want) / tol).max()
        assert worst <= 1, (tok, ctx.shape[1], worst)
        assert np.all(out[tok, c["heads"] * D:] == untouched)
    assert np.all(out[~seen] == untouched)  # padding and rows that are no decode tokens


def run_prefix(ops, c, hints=None, scratch=None, out=None, pools=None):
    shape = ops.attn_shape(c["heads"], c["kv_heads"], c["D"], c["bs"], q_stride=c["q"].shape[1], o_stride=c["o_stride"])
    meta = ops.TokenMeta.from_host(c["pos"], c["seq"], c["table_off"], c["tables"])
    if out is None:
        out = torch.full((len(c["pos"]), c["o_stride"]), 7.0, dtype=torch.float16, device="cuda")
    k, v = pools or (dev(c["k"]), dev(c["v"]))
    most = hints or (c["max_prefix"], c["max_suffix"])
    ops.shared_prefix_attention(shape, dev(c["q"]), meta, dev(c["tokens"]), dev(c["off"]), dev(c["lens"]), *most, k, v, out, scratch)
    torch.cuda.synchronize()
    assert ops.gemm_status() == 0  # no bounded pipeline wait gave up
    return out.cpu().numpy()


# Lengths for the plan behind which no prefix is short enough to be read as each token's own, and is split into slices of
# 128 keys; and more padding than tokens, behind which its slices are few.
SHARED = (1 << 20, 0)


def padded(c, entries=3000):
    return dict(c, tokens=np.concatenate([c["tokens"], np.full(entries, -1, np.int32)]))


PREFIX_CASES = [
    # D, heads, kv_heads, bs, groups
    (128, 32, 8, 16, [(500, [1, 7, 16, 40])]),
    (128, 32, 8, 16, [(4096, [1 + 37 * i for i in range(32)])]),
    (128, 32, 8, 16, [(1, [1]), (15, [1, 2]), (16, [16, 0]), (17, [1, 15, 16, 17])]),
    (128, 32, 8, 16, [(127, [3] * 5), (128, [3] * 33), (129, [0, 1, 130])]),
    (128, 40, 8, 16, [(5003, [20, 300, 1]), (0, [1, 200]), (1000, [5])]),
    (128, 8, 8, 32, [(333, [9] * 130)]),                       # one head to a KV head, more than one row tile
    (128, 16, 1, 16, [(2111, [4, 70, 500, 1])]),               # 16 heads to a KV head
    (128, 12, 4, 48, [(1000, [40, 7])]),                       # block size not a power of two
    (64, 14, 2, 32, [(5003, [1, 901, 33]), (17, [5] * 20), (640, [64])]),
    (64, 16, 16, 64, [(777, [1, 2, 3, 100, 64, 63])]),
    (64, 8, 2, 16, [(16384, [1000, 3])]),
    (64, 12, 4, 1, [(70, [1, 30]), (3, [4])]),                 # block size 1
    (64, 6, 2, 8, [(150, [5, 29, 77])]),                       # block size below the 16-key tile
    (64, 9, 3, 24, [(150, [5, 29, 77])]),
    (32, 16, 4, 8, [(777, [1, 100, 50]), (300, [12] * 24)]),
    (32, 32, 2, 16, [(600, [33, 1])]),
    (16, 4, 2, 16, [(53, [1, 2, 300]), (512, [17])]),
    (16, 4, 2, 16, [(40 + i, [1 + i % 5] * (1 + i % 3)) for i in range(45)]),   # more groups than a warp has lanes
    (128, 32, 8, 16, [(300, [-299, 5, -1, -150, 2000])]),      # contexts that end inside the prefix; the first has one key
    (128, 32, 8, 16, [(300, [5, -299, -1, -150, -300])]),      # and one without any key
    (64, 8, 2, 16, [(300, [None, 5, None, 9]), (100, [None]), (64, [3, None])]),  # padding
    (128, 8, 2, 16, [(0, [1, 5000])]),                         # nothing shared, long own contexts
    (64, 4, 4, 16, [(0, [1])]),
    (128, 4, 1, 16, [(40000, [2500])]),
    # few tokens behind a prefix of many slices, no long own part
    (128, 4, 1, 16, [(40000, [100, 7])]),
    (64, 16, 1, 16, [(9000, [3, None, -8990, 60, -8001]), (2, [1])]),
    (32, 8, 1, 8, [(20000, [90, 1]), (5, [5])]),
    (16, 4, 1, 16, [(8200, [1, 120, -8200])]),
]


@pytest.mark.parametrize("D,heads,kv_heads,bs,groups", PREFIX_CASES)
def test_shared_prefix_attention(ops, D, heads, kv_heads, bs, groups):
    c = prefix_case(D + len(groups), D, heads, kv_heads, bs, groups)
    out = run_prefix(ops, c)
    check_prefix(c, out, 7.0)
    assert np.array_equal(out, run_prefix(ops, c))  # the same bits on every run


@pytest.mark.parametrize("slices", ["many", "few"])
@pytest.mark.parametrize("D,heads,kv_heads,bs,groups", PREFIX_CASES)
def test_shared_prefix_attention_read_as_shared(ops, D, heads, kv_heads, bs, groups, slices):
    c = prefix_case(D + len(groups), D, heads, kv_heads, bs, groups)
    run = (lambda: run_prefix(ops, c, SHARED)) if slices == "many" else (lambda: run_prefix(ops, padded(c)))
    out = run()
    check_prefix(c, out, 7.0)
    assert np.array_equal(out, run())


@pytest.mark.parametrize("hints", [None, SHARED])
@pytest.mark.parametrize("D,heads,kv_heads,bs", [(128, 32, 8, 16), (64, 10, 2, 16), (32, 8, 2, 16), (16, 16, 1, 8)])
def test_shared_prefix_attention_with_peaked_scores_wide_rows_and_unrounded_queries(ops, D, heads, kv_heads, bs, hints):
    # queries three times wider than N(0,1), not representable in fp16: row maxima keep growing behind the first tile
    c = prefix_case(3, D, heads, kv_heads, bs, [(1500, [1, 40, 333]), (260, [600, 2])], peaked=3.0, q_pad=20, o_pad=24, dtype_q=np.float32)
    check_prefix(c, run_prefix(ops, c, hints), 7.0)
    if hints:
        check_prefix(c, run_prefix(ops, padded(c)), 7.0)


@pytest.mark.parametrize("hints", [(1, 1), (100000, 100000), (1 << 30, 0)])
@pytest.mark.parametrize("D,bs", [(128, 16), (32, 8)])
def test_shared_prefix_lengths_given_to_the_plan_do_not_change_the_result(ops, D, bs, hints):
    c = prefix_case(4, D, 8, 2, bs, [(1000, [1, 700, 33]), (20, [5, 6])])
    check_prefix(c, run_prefix(ops, c, hints), 7.0)


def test_shared_prefix_attention_without_a_shared_part(ops):
    c = prefix_case(6, 128, 8, 2, 16, [(200, [5, 40])])
    check_prefix(c, run_prefix(ops, c, (0, 240)), 7.0)  # max_prefix 0: every key is read as the token's own


@pytest.mark.parametrize("D,heads,kv_heads,bs", [(128, 32, 8, 16), (64, 8, 8, 8)])
def test_shared_prefix_attention_agrees_with_decode_attention(ops, D, heads, kv_heads, bs):
    c = prefix_case(8, D, heads, kv_heads, bs, [(700, [1, 30, 200]), (90, [9, 600])])
    got = run_prefix(ops, c).astype(np.float32)
    shape = ops.attn_shape(heads, kv_heads, D, bs)
    meta = ops.TokenMeta.from_host(c["pos"], c["seq"], c["table_off"], c["tables"])
    out = torch.zeros((len(c["pos"]), heads * D), dtype=torch.float16, device="cuda")
    ops.decode_attention(shape, dev(c["q"]), meta, dev(c["tokens"]), 900, dev(c["k"]), dev(c["v"]), out)
    want = out.cpu().numpy().astype(np.float32)[c["tokens"]]
    # two kernels, each within the bound of check_prefix
    assert np.abs(got[c["tokens"]] - want).max() <= 4 * (H16 + 2.0 ** -15) * np.abs(c["v"][~np.isnan(c["v"])].astype(np.float32)).max()


@pytest.mark.parametrize("hints", [None, SHARED])
@pytest.mark.parametrize("D,bs", [(128, 16), (32, 8)])
def test_shared_prefix_attention_of_a_padded_batch(ops, D, bs, hints):
    # entries before the first group and behind the last are padding, whatever they name
    c = prefix_case(12, D, 8, 2, bs, [(300, [5, 40]), (17, [1, 2, 3])])
    c["tokens"] = np.concatenate([[c["tokens"][1], -1], c["tokens"], [c["tokens"][0]] * 3]).astype(np.int32)
    c["off"] = c["off"] + 2
    out = run_prefix(ops, c, hints)
    c["tokens"], c["off"] = c["tokens"][2:-3], c["off"] - 2
    check_prefix(c, out, 7.0)


@pytest.mark.parametrize("hints", [None, SHARED])
def test_shared_prefix_attention_of_the_same_row_twice(ops, hints):
    c = prefix_case(13, 64, 8, 2, 16, [(300, [5, 40, 7])])
    want = run_prefix(ops, c, hints)
    c["tokens"], c["off"] = np.concatenate([c["tokens"], c["tokens"][:1]]), np.asarray([0, 4], np.int32)
    assert np.array_equal(run_prefix(ops, c, hints), want)  # one group: either result has the same bits


@pytest.mark.parametrize("hints", [(3000, 30), SHARED])
def test_shared_prefix_attention_scratch_may_hold_anything(ops, hints):
    c = prefix_case(9, 128, 8, 2, 16, [(3000, [1, 30]), (0, [9]), (100, [4])])
    shape = ops.attn_shape(8, 2, 128, 16)
    need = ops.shared_prefix_scratch_bytes(shape, 4, 3, *hints)
    scratch = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")  # NaN in every word
    check_prefix(c, run_prefix(ops, c, hints, scratch=scratch[:need]), 7.0)
    assert torch.all(scratch[need:] == 255)


CAPTURE_AFTER_A_SMALL_CALL = """
import torch
from relay_b200 import ops
i32 = dict(dtype=torch.int32, device="cuda")
shape = ops.attn_shape(8, 2, 64, 16)
pool = torch.randn(40, 2, 16, 64, device="cuda").half()
q = torch.randn(1, 12 * 64, device="cuda")
meta = ops.TokenMeta(torch.tensor([599], **i32), torch.tensor([0], **i32), torch.tensor([0], **i32), torch.arange(40, **i32))
args = shape, q, meta, torch.tensor([0], **i32), torch.tensor([0, 1], **i32), torch.tensor([590], **i32)
outs = [torch.zeros(1, 512, dtype=torch.float16, device="cuda") for _ in range(2)]
ops.shared_prefix_attention(*args, 590, 10, pool, pool, outs[0])
scratch = torch.empty(ops.shared_prefix_scratch_bytes(shape, 1, 1, 1 << 20, 0), dtype=torch.uint8, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.shared_prefix_attention(*args, 1 << 20, 0, pool, pool, outs[1], scratch)
graph.replay()
torch.cuda.synchronize()
assert (outs[0].float() - outs[1].float()).abs().max() <= (2.0 ** -9 + 2.0 ** -14) * pool.float().abs().max()
"""


def test_shared_prefix_attention_captured_after_a_small_call(ops):
    # in a process of its own: the small call is the device's first, and takes other kernels than the captured one
    subprocess.run([sys.executable, "-c", CAPTURE_AFTER_A_SMALL_CALL], check=True, timeout=300,
                   cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


@pytest.mark.parametrize("D", [128, 32])
def test_page_offsets_past_32_bits(ops, D):
    # a pool of more than 2^31 values, the batch's pages at its far end; the append and the attention both go there
    heads, kv_heads, bs = 8, 2, 16
    c = prefix_case(10, D, heads, kv_heads, bs, [(300, [5, 40]), (17, [1])])
    per = kv_heads * bs * D
    shift = (1 << 31) // per + 8
    nb = shift + len(c["k"])
    pools = []
    for name in ("k", "v"):
        pool = torch.empty((nb, kv_heads, bs, D), dtype=torch.float16, device="cuda")
        pool[shift:] = dev(c[name])
        pools.append(pool)
    c["tables"] = (c["tables"] + shift).astype(np.int32)
    for hints in (None, SHARED):
        check_prefix(c, run_prefix(ops, c, hints, pools=pools), 7.0)
    qkv = torch.randn(1, (heads + 2 * kv_heads) * D, device="cuda")
    meta = ops.TokenMeta.from_host([3], [0], [0], [nb - 1])
    ops.qkv_norm_post(qkv, None, None, None, 1e-6, torch.ones(D // 2, device="cuda"), meta, qkv, *pools, heads, kv_heads, D, bs)
    assert torch.equal(pools[1][nb - 1, :, 3].flatten(), qkv[0, (heads + kv_heads) * D:].half())


# ---- logits ------------------------------------------------------------------------------------


def adjust_f64(x, pen, history, history_len, prompt_len, bias_ids, bias_values, bias_len, mask):
    """(float64 result, the magnitude its rounding errors refer to)."""
    y = x.astype(np.float64)
    R, V = y.shape
    reach = np.abs(y)
    with np.errstate(invalid="ignore"):
        for r in range(R):
            if pen is not None:
                rep, pres, freq = (float(a) for a in pen[r][:3])
                n = max(0, min(int(history_len[r]), history.shape[1]))
                p = 0 if prompt_len is None else max(0, min(int(prompt_len[r]), n))
                ids, gen = history[r, :n].astype(np.int64), history[r, p:n].astype(np.int64)
                seen = np.bincount(ids[(ids >= 0) & (ids < V)], minlength=V) > 0
                count = np.bincount(gen[(gen >= 0) & (gen < V)], minlength=V).astype(np.float64)
                y[r] = np.where(seen, np.where(y[r] > 0, y[r] / rep, y[r] * rep), y[r])
                reach[r] = np.maximum(reach[r], np.abs(y[r])) + count * abs(freq) + (count > 0) * abs(pres)
                y[r] -= np.where(count > 0, count * freq + pres, 0)
            if bias_ids is not None:
                n = max(0, min(int(bias_len[r]), bias_ids.shape[1]))
                last = {int(i): float(b) for i, b in zip(bias_ids[r, :n], bias_values[r, :n]) if 0 <= i < V}
                for i, b in last.items():
                    y[r, i] += b
                    reach[r, i] += abs(b)
            if mask is not None:
                bits = np.unpackbits(mask[r].view(np.uint8), bitorder="little")[:V]
                y[r, bits == 0] = -np.inf
    return y, reach


def check_logits(got, want, reach):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf].astype(np.float32)) and np.all(np.isfinite(got) == np.isfinite(want))
    ok = np.isfinite(want)
    # the quotient or product, frequency * count, + presence, the difference and the bias: at most 5 roundings
    assert np.all(np.abs(got[ok] - want[ok]) <= 5 * U32 * reach[ok] + 1e-37)


LOGIT_CASES = [
    # rows, vocab, history columns, bias columns, mask
    (1, 128256, 800, 4, True),
    (3, 128256, 5000, 300, True),
    (7, 32000, 40, 0, False),
    (5, 1000, 64, 5, True),
    (2, 31, 9, 3, True),
    (4, 33, 9, 3, True),
    (1, 1, 2, 1, True),
    (9, 4097, 4096, 64, True),
    (300, 513, 33, 1, True),
    (2, 151937, 20000, 7, True),
    (3, 5000, 0, 0, True),
    (3, 5000, 12, 0, False),
    (2, 300000, 50000, 1000, True),
    # batches whose segments are long: of 4096, of 8192 and of 16384 tokens
    (6, 128256, 900, 3, True),
    (5, 151937, 900, 0, False),
    (100, 33000, 700, 3, True),
    (48, 128256, 3000, 16, True),
    (40, 151937, 5000, 0, False),
    (300, 20000, 60, 2, True),
    (64, 128256, 3000, 16, True),
    (64, 151937, 300, 40, True),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R,V,hist,biases,use_mask", LOGIT_CASES)
def test_adjust_logits(ops, R, V, hist, biases, use_mask, in_place):
    rng = np.random.Generator(np.random.PCG64(V + R))
    x = (rng.standard_normal((R, V)) * 4).astype(np.float32)
    x[0, ::7] = 0.0
    x[0, ::11] = -np.inf
    x[R - 1, ::13] = np.nan
    pen = np.stack([1 + rng.random(R), rng.random(R) * 2 - 0.5, rng.random(R) - 0.3, np.zeros(R)], 1).astype(np.float32)
    history = (rng.random((R, hist)) ** 3 * V).astype(np.int32)  # frequent and rare tokens
    if hist:
        history[:, ::5] = history[:, :1]  # one token many times over
        history[rng.random(history.shape) < 0.05] = rng.choice(np.asarray([-1, -2 ** 31, V, 2 ** 31 - 1], np.int32))
    history_len = rng.integers(0, hist + 1, R).astype(np.int32)
    history_len[0] = hist + 7  # counts as the whole row
    if R > 1:
        history_len[1] = -3
    prompt_len = rng.integers(0, hist + 3, R).astype(np.int32)
    bias_ids = bias_values = bias_len = mask = None
    if biases:
        bias_ids = rng.integers(0, V, (R, biases)).astype(np.int32)
        bias_ids[:, -1] = bias_ids[:, 0]  # the same token twice
        bias_ids[0, biases // 2] = V
        bias_values = (rng.standard_normal((R, biases)) * 5).astype(np.float32)
        bias_len = rng.integers(0, biases + 1, R).astype(np.int32)
        bias_len[R - 1] = biases
    if use_mask:
        mask = rng.integers(0, 2 ** 32, (R, (V + 31) // 32 + 1), dtype=np.uint32).view(np.int32)
        mask[0] = 0  # leaves nothing
        mask[R // 2] |= 1
    opt = lambda a: None if a is None else dev(a)  # noqa: E731
    wide = torch.full((R, V + 3), 3.0, device="cuda")
    wide[:, :V] = dev(x)
    logits = wide[:, :V]
    out = logits if in_place else torch.full((R, V), 5.0, device="cuda")
    ops.adjust_logits(logits, out, dev(pen), dev(history), dev(history_len), dev(prompt_len), opt(bias_ids), opt(bias_values),
                      opt(bias_len), opt(mask))
    want, reach = adjust_f64(x, pen, history, history_len, prompt_len, bias_ids, bias_values, bias_len, mask)
    check_logits(out.cpu().numpy(), want, reach)
    assert torch.all(wide[:, V:] == 3)
    if not in_place:
        assert np.array_equal(logits.cpu().numpy(), x, equal_nan=True)
    elif use_mask:
        tok = torch.empty(R, dtype=torch.int32, device="cuda")
        ops.argmax_rows(out.contiguous(), tok)
        assert R == 1 or tok[0].item() == 0  # the row whose mask leaves nothing (a single row keeps some tokens)


@pytest.mark.parametrize("part", ["nothing", "penalties", "no prompt", "bias", "mask"])
def test_adjust_logits_parts_alone(ops, part):
    rng = np.random.Generator(np.random.PCG64(3))
    R, V = 4, 9001
    x = rng.standard_normal((R, V)).astype(np.float32)
    pen = np.asarray([[1.3, 0.5, 0.25, 0]] * R, np.float32)
    history = rng.integers(0, V, (R, 500)).astype(np.int32)
    lens, prompt = np.full(R, 500, np.int32), np.full(R, 250, np.int32)
    ids, values, bl = history[:, :20].copy(), rng.standard_normal((R, 20)).astype(np.float32), np.full(R, 20, np.int32)
    mask = rng.integers(0, 2 ** 32, (R, (V + 31) // 32), dtype=np.uint32).view(np.int32)
    args = dict(penalties=None, history=None, history_len=None, prompt_len=None, bias_ids=None, bias_values=None, bias_len=None, mask=None)
    if part in ("penalties", "no prompt"):
        args |= dict(penalties=pen, history=history, history_len=lens, prompt_len=prompt if part == "penalties" else None)
    elif part == "bias":
        args |= dict(bias_ids=ids, bias_values=values, bias_len=bl)
    elif part == "mask":
        args |= dict(mask=mask)
    out = torch.empty((R, V), device="cuda")
    ops.adjust_logits(dev(x), out, **{k: None if v is None else dev(v) for k, v in args.items()})
    want, reach = adjust_f64(x, *args.values())
    check_logits(out.cpu().numpy(), want, reach)
    if part == "nothing":
        assert np.array_equal(out.cpu().numpy(), x)


def test_adjust_logits_row_offsets_past_32_bits(ops):
    R, V = 4, 40000
    ld = (1 << 31) // 2  # the third row starts 2^31 values in
    big = torch.empty(3 * ld + V, device="cuda")
    view = big.as_strided((R, V), (ld, 1))
    x = np.random.Generator(np.random.PCG64(1)).standard_normal((R, V)).astype(np.float32)
    view.copy_(dev(x))
    mask = np.full((R, V // 32), 0x0F0F0F0F, np.int32)
    ops.adjust_logits(view, view, mask=dev(mask))
    want, reach = adjust_f64(x, None, None, None, None, None, None, None, mask)
    check_logits(view.cpu().numpy(), want, reach)


# ---- together ----------------------------------------------------------------------------------


class Step:
    """One layer's attention and the sampler of a decode step: 12 requests behind two prompts, one slot of
    the batch unused, under penalties and a grammar; every buffer stays where it is between steps."""

    def __init__(self, ops, seed, lengths):
        self.ops, self.lengths = ops, lengths
        rng = np.random.Generator(np.random.PCG64(seed))
        self.heads, self.kv_heads, self.D, self.bs, self.V = 16, 4, 64, 16, 2000
        self.c = c = prefix_case(seed, self.D, self.heads, self.kv_heads, self.bs,
                                 [(333, [1 + 9 * i for i in range(7)]), (64, [1, 2, 30, 64]), (0, [77])])
        n = len(c["tokens"])
        self.T = T = n + 1  # the last batch row is padding
        order = c["tokens"]
        self.rows = np.arange(n, dtype=np.int32)
        self.pos = np.full(T, -1, np.int32)
        self.seq = np.full(T, -1, np.int32)
        self.pos[:n], self.seq[:n] = c["pos"][order], c["seq"][order]
        self.qkv = rng.standard_normal((T, (self.heads + 2 * self.kv_heads) * self.D)).astype(np.float32)
        self.qn, self.kn = ((1 + 0.1 * rng.standard_normal(self.D)).astype(np.float32) for _ in range(2))
        self.inv = (10000.0 ** -(np.arange(0, self.D, 2) / self.D)).astype(np.float32)
        self.head = (rng.standard_normal((self.V, self.heads * self.D)) * 0.2).astype(np.float32)
        self.pen = np.asarray([[1.2, 0.3, 0.2, 0]] * T, np.float32)
        self.history = rng.integers(0, self.V, (T, 50)).astype(np.int32)
        self.history_len, self.prompt_len = np.full(T, 50, np.int32), np.full(T, 20, np.int32)
        self.mask = rng.integers(0, 2 ** 32, (T, (self.V + 31) // 32), dtype=np.uint32).view(np.int32)
        g = {k: dev(getattr(self, k)) for k in ("qkv", "qn", "kn", "inv", "head", "pen", "history", "history_len", "prompt_len", "mask")}
        self.g = g
        self.meta = ops.TokenMeta.from_host(self.pos, self.seq, c["table_off"], c["tables"])
        self.tokens = dev(np.concatenate([self.rows, [-1]]).astype(np.int32))
        self.off, self.lens = dev(c["off"]), dev(c["lens"])
        self.k, self.v = dev(np.nan_to_num(c["k"])), dev(np.nan_to_num(c["v"]))
        self.shape = ops.attn_shape(self.heads, self.kv_heads, self.D, self.bs, q_stride=self.heads * self.D)
        self.q = torch.zeros((T, self.heads * self.D), device="cuda")
        self.out = torch.zeros((T, self.heads * self.D), dtype=torch.float16, device="cuda")
        self.logits = torch.zeros((T, self.V), device="cuda")
        self.picked = torch.full((T,), -1, dtype=torch.int32, device="cuda")
        self.sampling = torch.zeros((T, 32), dtype=torch.uint8, device="cuda")  # temperature 0
        self.scratch = torch.empty(ops.shared_prefix_scratch_bytes(self.shape, T, 3, *lengths), dtype=torch.uint8, device="cuda")

    def run(self):
        g, o = self.g, self.ops
        o.qkv_norm_post(g["qkv"], None, g["qn"], g["kn"], 1e-5, g["inv"], self.meta, self.q, self.k, self.v, self.heads, self.kv_heads,
                        self.D, self.bs)
        o.shared_prefix_attention(self.shape, self.q, self.meta, self.tokens, self.off, self.lens, *self.lengths, self.k, self.v, self.out,
                                  self.scratch)
        torch.mm(self.out.float(), g["head"].t(), out=self.logits)
        o.adjust_logits(self.logits, self.logits, g["pen"], g["history"], g["history_len"], g["prompt_len"], mask=g["mask"])
        o.sample_rows(self.logits, self.sampling, self.picked)

    def check(self):
        n = self.T - 1
        q, k, v, _ = norm_rope_f64(self.g["qkv"].cpu().numpy()[:n], None, self.qn, self.kn, 1e-5, self.inv, self.pos[:n], self.heads,
                                   self.kv_heads, self.D, self.D)
        contexts = []
        for i, ctx in enumerate(self.c["contexts"]):  # the step's own key and value are the last of the context
            page = int(self.c["tables"][self.c["table_off"][self.seq[i]] + self.pos[i] // self.bs])
            new_k, new_v = (pool[page, :, int(self.pos[i]) % self.bs].cpu().numpy() for pool in (self.k, self.v))
            assert np.all(np.abs(new_k - k[i]) <= H16 * np.abs(k[i]) + 2.0 ** -25 + NORM_TOL * 2 * np.abs(k).max())
            assert np.array_equal(new_v, v[i].astype(np.float16))
            ctx = ctx.copy()
            ctx[0, -1], ctx[1, -1] = new_k, new_v
            contexts.append(ctx)
        case = dict(self.c, tokens=self.rows, contexts=contexts, q=self.q.cpu().numpy())
        assert np.all(np.abs(case["q"][:n].reshape(q.shape) - q) <= NORM_TOL * 2 * np.abs(q).max())
        check_prefix(case, self.out.cpu().numpy(), 0.0)
        raw = self.out.float() @ self.g["head"].t()
        want, reach = adjust_f64(raw.cpu().numpy(), self.pen, self.history, self.history_len, self.prompt_len, None, None, None, self.mask)
        got = self.logits.cpu().numpy()
        check_logits(got, want, reach)
        assert self.picked.cpu().tolist() == [oracle.argmax(r) for r in got]


LENGTHS = [(333, 77), SHARED]


@pytest.mark.parametrize("lengths", LENGTHS)
def test_a_decode_step_of_all_three_operators(ops, lengths):
    s = Step(ops, 21, lengths)
    s.run()
    torch.cuda.synchronize()
    s.check()


@pytest.mark.parametrize("lengths", LENGTHS)
def test_a_decode_step_replayed_as_a_graph_follows_its_inputs(ops, lengths):
    s = Step(ops, 22, lengths)
    s.run()  # attributes are set once per device
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        s.g["qkv"].copy_(torch.randn(s.g["qkv"].shape, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        s.check()
        graphed = [t.clone() for t in (s.q, s.out, s.logits, s.picked)]
        s.run()
        torch.cuda.synchronize()
        for a, b in zip(graphed, (s.q, s.out, s.logits, s.picked)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("lengths", LENGTHS)
def test_two_decode_steps_at_once_on_two_streams(ops, lengths):
    steps = [Step(ops, 23, lengths), Step(ops, 24, lengths)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.run()
    torch.cuda.synchronize()
    for s in steps:
        s.check()
