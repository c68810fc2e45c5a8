"""What the decode step's operators promise about order, odd values and reports,
on the GPU, against plain forms in Python integers and float64."""
import pytest
import torch

import q3s

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda_device):
    q3s.load_torch_ops()
    return cuda_device


# ---- order of calls -----------------------------------------------------------

def exact_product(a, a_s, w, w_s):
    """(values, tolerance) of an fp32 8-bit product: an exact sum, its conversion and two products, each off by 2^-24."""
    want = (a.double() @ w.double().t()) * a_s.double()[:, None] * w_s.double()
    return want, 2.0 ** -22 * want.abs()


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 40])
def test_returned_values_as_the_next_weight(dev, rows):
    """The values that a one-launch Linear writes are the weight of the product right behind it."""
    g = torch.Generator(device=dev).manual_seed(rows)
    w = torch.randint(-127, 128, (2048, 2048), device=dev, generator=g, dtype=torch.int8)
    ws = torch.rand(2048, device=dev, generator=g) + 0.5
    for _ in range(10):
        x = torch.randn(rows, 2048, device=dev, generator=g).bfloat16()
        torch.cuda.synchronize()
        _, v, s = q3s.int8_linear(x, w, ws, return_quantized=True)
        z = q3s.int8_matmul(v, s, v, s, dtype=torch.float32)
        want, tol = exact_product(v, s, v, s)
        assert bool(((z.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("rows", [1, 8, 40, 300])
def test_weight_written_by_another_kernel_right_before(dev, rows):
    g = torch.Generator(device=dev).manual_seed(rows)
    a = torch.randint(-127, 128, (rows, 2048), device=dev, generator=g, dtype=torch.int8)
    s = torch.rand(5000, device=dev, generator=g) + 0.5
    w = torch.empty(5000, 2048, device=dev, dtype=torch.int8)
    for _ in range(5):
        fresh = torch.randint(-127, 128, (5000, 2048), device=dev, generator=g, dtype=torch.int8)
        torch.cuda.synchronize()
        torch.add(fresh, 0, out=w)
        y = q3s.int8_matmul(a, s[:rows], w, s, dtype=torch.float32)
        want, tol = exact_product(a, s[:rows], fresh, s)
        assert bool(((y.double() - want).abs() <= tol).all())
