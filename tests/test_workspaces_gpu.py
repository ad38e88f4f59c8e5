"""Workspaces that calls share: linears of several sizes on one stream, graphs whose stream
went on to larger calls, and paged forward passes on several streams and in graphs."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(cuda):
    import torch as _t
    return _t


@pytest.fixture(scope="module")
def lib(cuda):
    import dial_cuda
    return dial_cuda


@pytest.fixture(autouse=True)
def no_device_error(cuda):
    import dial_cuda
    yield
    assert dial_cuda.lib().dial_device_error(1) == 0, "a kernel reported an error"


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("qtype", ["Q4_0", "Q8_0"])
@pytest.mark.parametrize("K", [512, 1152, 2080])
@pytest.mark.parametrize("M", [1, 9])
def test_gguf_linears_of_several_sizes_on_one_stream(torch, lib, qtype, K, M):
    """A linear with few outputs between two calls of one with many: the same bits each time."""
    g = gen(torch, K + M)
    lins = [lib.GgufLinear.quantize(torch.randn((N, K), generator=g, device="cuda") * 0.05, getattr(lib, qtype))
            for N in (2048, 512, 1024, 16)]
    x = torch.randn((M, K), generator=g, device="cuda").half()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        want = [l.forward(x) for l in lins]
        for _ in range(3):
            for i in (0, 1, 3, 2, 0):
                got = lins[i].forward(x)
                side.synchronize()
                assert torch.equal(got, want[i]), i
    for l, y in zip(lins, want):
        ref = x.double() @ l.dequantize(torch.float32).double().T
        # the activations' Q8_0 rounding: half a step of absmax / 127 a value
        bound = (x.abs().amax(-1, keepdim=True).double() / 254 * 1.01) * l.dequantize(torch.float32).double().abs().sum(-1) + 2.0 ** -11 * ref.abs() + 1e-6
        assert torch.all((y.double() - ref).abs() <= bound)
