"""The decode-step operators around a shared prompt in the forms that test_gpu_step_ops.py does not reach."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_gpu_step_ops import NORM_TOL, dev, norm_rope_f64, ops  # noqa: E402, F401


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
