"""The rotary append with head counts that leave a warp of the kernel half occupied."""
import numpy as np
import pytest

from test_serve_gpu import HD, PAGE, _t, appended, assert_half

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("hq,hkv", [(15, 1), (7, 7), (47, 1), (33, 32), (95, 1), (1, 24)])
def test_append_of_an_odd_number_of_heads(ctx, hq, hkv, norm):
    rng = np.random.default_rng(hq)
    t, pages, width = 9, 4, (hq + 2 * hkv) * HD
    x = rng.standard_normal((t, width), dtype=np.float32)
    pos = rng.integers(0, 5000, t).astype(np.int32)
    slots = rng.permutation(pages * PAGE)[:t].astype(np.int32)
    qg, kg = (1 + 0.2 * rng.standard_normal((2, HD))).astype(np.float32) if norm else (None, None)
    pool = ctx.kv_pool(pages, hkv)
    pool.tensor().zero_()
    gains = dict(q_gain=_t(qg), k_gain=_t(kg)) if norm else {}
    q = ctx.rope_append(pool, _t(x), _t(pos), _t(slots), 1e4, eps=1e-6, **gains)
    q_want, want = appended(x, pos, slots, 1e4, hq, hkv, qg, kg, 1e-6, np.zeros((pages, hkv, 2, PAGE, HD)))
    size = 8.0 * (1.8 if norm else 1.0)
    assert_half(q.cpu().numpy(), q_want, size, 5000)
    assert_half(pool.tensor().cpu().numpy(), want, size, 5000)
    pool.free()
    ctx.device_status()
