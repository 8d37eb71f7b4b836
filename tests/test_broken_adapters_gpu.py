"""Requests beside one whose adapter is broken (its b holds NaN or infinities):
long contractions, and what the repair of their rows costs."""
import pytest
import torch

from tests import block_ops_support as sup
from tests.test_block_ops_gpu import _gen, _lora_inputs

pytestmark = pytest.mark.gpu


# pairs of SMs (ranks of one and of two K blocks) and token columns; contractions
# and outputs that no block or vector divides
@pytest.mark.parametrize("N,K,M,r", [(600, 4104, 520, 16), (300, 6150, 264, 80), (200, 4104, 260, 64),
                                     (40, 8203, 133, 12), (3, 4099, 70, 40)])
def test_requests_beside_an_adapter_that_is_nan_throughout(N, K, M, r):
    from foundry_trainer_b200 import ops
    g = _gen(N + K)
    ld = (K + 7) // 8 * 8  # rows on 16 bytes; what lies between them is not read
    x, w, a, b, bias = _lora_inputs(g, N, ld, M, r, True, 4)
    for t in (x, w, a):
        t[..., K:] = float("nan")
    x, w, a = x[:, :K], w[:, :K], a[:, :, :K]
    scales = torch.rand(4, generator=g, device="cuda") + 0.5
    ids = torch.tensor([0, 3, -1, 1, 0, 2, 0], device="cuda")[torch.arange(N, device="cuda") % 7]
    ids = ids.to(torch.int32)
    b[3] = float("nan")
    b[2, 5] = float("inf")
    got = ops.lora_linear_many(x, w, a, b, ids, scales, bias=bias)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for e in (0, 1, -1):
        rows = ids == e
        if not rows.any():
            continue
        gain = scales[e].item() if e >= 0 else 0.0
        want, tol, _, _ = sup.lora_ref(x[rows].double(), w.double(), a[max(e, 0)].double(),
                                       b[max(e, 0)].double(), gain, bias.double())
        sup.within(got[rows], want, tol, f"adapter {e}")
    assert torch.isnan(got[ids == 3]).all()


@pytest.mark.parametrize("N", [600, 200])
def test_the_repair_is_of_the_order_of_the_call(N):
    # Beside an adapter that is NaN throughout every value of the other rows is
    # multiplied again, by four warps a tile in place of the tensor memory's
    # products: an order of magnitude of time, not three or four (a scalar sum a
    # value). The bound of 100 calls lies between.
    from foundry_trainer_b200 import ops
    g = _gen(21)
    x, w, a, b, _ = _lora_inputs(g, N, 4096, 1024, 16, False, 3)
    scales = torch.ones(3, device="cuda")
    ids = (torch.arange(N, device="cuda") % 3).to(torch.int32)
    broken = b.clone()
    broken[1] = float("nan")

    def best(f):
        times = []
        for _ in range(4):
            t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            t0.record()
            f()
            t1.record()
            torch.cuda.synchronize()
            times.append(t0.elapsed_time(t1))
        return min(times)

    clean = best(lambda: ops.lora_linear_many(x, w, a, b, ids, scales))
    slow = best(lambda: ops.lora_linear_many(x, w, a, broken, ids, scales))
    assert slow <= 100 * clean, (slow, clean)
