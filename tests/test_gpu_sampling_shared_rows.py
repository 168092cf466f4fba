"""Every way in which workgroups take rows of logits, against the rules worked out in 64 bits."""
import pytest
import torch

from test_gpu_sampling import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,V,dtype", [(17, 28000, torch.float16), (64, 30011, torch.bfloat16), (33, 131072, torch.float32), (65, 28001, torch.float32),
                                       (128, 30001, torch.float16), (130, 28003, torch.bfloat16), (140, 50272, torch.float32), (20, 27999, torch.float16)])
def test_rows_shared_by_any_number_of_workgroups(gpu_device, R, V, dtype):
    """17 to 64 rows of 28000 and more go to four workgroups each, 65 to 128 to two, more to one; as many tokens counted as are counted in the first
    pass (256) or not, whole rows, targets in the tail."""
    gen = torch.Generator(device=gpu_device).manual_seed(R + V)
    logits = torch.randn((R, V), generator=gen, device=gpu_device) * 2.5
    logits[:, ::701] += 4
    logits[1] = 0.5
    logits[2, :-3] = float("-inf")
    logits[3, ::2] = float("nan")
    logits = logits.to(dtype)
    cycle = lambda values: [values[r % len(values)] for r in range(R)]
    u = torch.rand(R, generator=gen, device=gpu_device).tolist()
    check(logits, u, 1.0)
    check(logits, u, cycle([1.0, 0.8, 1.5, 0.0, 3.0]), cycle([255, 256, 257, 3000, 0, 1, V - 1]), cycle([1.0, 0.9, 0.999, 0.5]), cycle([0.0, 0.01, 1e-5]))
    check(logits, cycle([1 - 2.0 ** -24, 0.0, 0.999]), cycle([1.0, 2.0]), cycle([0, 20000]), cycle([0.9999, 1.0]))
