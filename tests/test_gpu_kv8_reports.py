"""What the 8-bit cache's kernels report: pages that do not exist, scales that cannot be, and who gets to know."""
import pytest
import torch

from pasa_b200 import ops
from test_gpu_kv8 import Pages, i32, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("queries", [1, 40, 200])
@pytest.mark.parametrize("bad", [0.3, 0.0, -1.0, -0.0, float("inf"), 2.0 ** -130])
def test_scales_of_keys_that_are_no_power_of_two(cuda_device, bad, queries):
    p = Pages([200, 100], 2, 64).fill()
    q, n = randn(2, 4, queries, 64), i32([200, 100])
    clean = ops.kv8_attention(q, p.cache, p.table, n)
    scales = p.cache.k_scale.clone()
    scales[p.rows[0][1], 1] = bad
    out = ops.kv8_attention(q, p.cache._replace(k_scale=scales), p.table, n)
    with pytest.raises(RuntimeError, match="power of two"):
        ops.check_operator_errors()
    assert out[0, 2:].isnan().all()
    assert torch.equal(out[0, :2], clean[0, :2]) and torch.equal(out[1], clean[1])
    out = ops.kv8_attention(q, p.cache._replace(k_scale=scales), p.table, i32([64, 100]))  # before that page
    assert out.isfinite().all()
    ops.check_operator_errors()


def test_a_scale_of_nan_is_a_page_with_nan(cuda_device):
    p = Pages([200], 1, 128).fill()
    p.cache.k_scale[p.rows[0][2]] = float("nan")
    assert ops.kv8_attention(randn(1, 2, 3, 128), p.cache, p.table, i32([200])).isnan().all()
    ops.check_operator_errors()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries", [1, 40, 200])
@pytest.mark.parametrize("at", [0, 3, 40])
def test_a_page_that_does_not_exist_reads_as_nan(cuda_device, dim, queries, at):
    """And not as what another request has in some page."""
    p = Pages([2700, 500], 2, dim).fill()
    q, n = randn(2, 2, queries, dim), i32([2700, 500])
    clean = ops.kv8_attention(q, p.cache, p.table, n)
    for bad in (-1, p.pages, 1 << 30, -(1 << 31)):
        table = p.table.clone()
        table[0, at] = bad
        out = ops.kv8_attention(q, p.cache, table, n)
        with pytest.raises(RuntimeError, match="page that does not exist"):
            ops.check_operator_errors()
        assert out[0].isnan().all() and torch.equal(out[1], clean[1])


def test_reports_of_another_stream_are_not_lost(cuda_device):
    """A kernel on one stream reports while another stream asks, over and over: somebody gets to know of each."""
    p = Pages([300], 1, 64).fill()
    table = p.table.clone()
    table[0, 4] = -1
    q, n = randn(1, 1, 3, 64), i32([300])
    torch.cuda.synchronize()
    ops.check_operator_errors()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(100):
        told = 0
        with torch.cuda.stream(one):
            ops.kv8_attention(q, p.cache, table, n)
            done = torch.cuda.Event()
            done.record()
        last = False
        with torch.cuda.stream(two):
            while not last:
                last = done.query()
                try:
                    ops.check_operator_errors()
                except RuntimeError:
                    told += 1
        assert told == 1
    with torch.cuda.stream(two):
        ops.check_operator_errors()
