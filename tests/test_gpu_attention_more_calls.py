"""Calls with first tokens and with shared prefixes that callers make now and then: batches that share nothing this step,
lengths that are only bounds, outputs without their log-sum-exp."""
import pytest

torch = pytest.importorskip("torch")
import attention_more_reference as more  # noqa: E402
from test_gpu_attention import Problem  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


@pytest.mark.parametrize("new", [1, 40])
def test_a_batch_that_shares_nothing(pkg, dev, new):
    p = Problem([new + 60, new + 75], [new] * 2, 2, 4, 128, 16, "f16")
    q, c, table, starts, kv_len = p.on(pkg, dev)
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    for path in (pkg.SHARED_AUTO, pkg.SHARED_ONCE, pkg.SHARED_EACH):
        out, lse = pkg.shared_attention(q, c, table, starts, kv_len, none, new, new + 75, 0, lse=True, scale=p.scale,
                                        path=path)
        more.compare(p, out.cpu(), lse.cpu(), more.window_and_sinks(True, 0, 0))
    with pytest.raises(pkg.Iq4xsError):
        pkg.shared_attention(q, c, table, starts, kv_len, none, new, new + 75, -1)
