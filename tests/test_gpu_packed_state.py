"""State dicts of the packed modules: a checkpoint with row-major scales gives the same results as one with tiles."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(native_lib):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    torch.cuda.set_device(0)
    return torch.device("cuda", 0)


def checkpoint(weight, layout):
    """What a packed module of the weight [.., N, K] saves, with its scales in `layout`."""
    import rtx_b200
    from rtx_b200.configs import MXFP8QuantConfig

    n, k = weight.numel() // weight.shape[-1], weight.shape[-1]
    dense = rtx_b200.MXFP8Linear(k, n, device=weight.device)
    with torch.no_grad():
        dense.weight.copy_(weight.reshape(n, k))
    return dense.to_quantized_weight(config=MXFP8QuantConfig(scale_layout=layout)).state_dict()


@pytest.mark.parametrize("layout", ["row_major", "mma128"])
def test_either_layout_loads(dev, layout):
    import rtx_b200

    torch.manual_seed(2)
    # both layouts of these scales have the same number of bytes
    w = (torch.randn(2, 128, 256, device=dev) * torch.logspace(-2, 2, 256, device=dev)).bfloat16()
    x = torch.randn(40, 256, device=dev).bfloat16()
    offsets = torch.tensor([0, 25, 40], dtype=torch.int32, device=dev)
    m = rtx_b200.MXFP8LinearEpilogue(256, 256, bias=False, activation="silu", device=dev).to_quantized_weight()
    m.load_state_dict(checkpoint(w, layout))
    want = rtx_b200.mxfp8_linear_epilogue(x, rtx_b200.quantize_mxfp8(w.view(256, 256)), activation="silu")
    assert torch.equal(m(x), want)
    assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x, m.packed_weight(), activation="silu"), want)
    g = rtx_b200.MXFP8GroupedLinear(2, 256, 128, device=dev).to_quantized_weight()
    g.load_state_dict(checkpoint(w, layout))
    want = rtx_b200.mxfp8_grouped_linear(x, rtx_b200.quantize_mxfp8(w), offsets)
    assert torch.equal(g(x, offsets), want)
    again = rtx_b200.MXFP8GroupedLinear(2, 256, 128, device=dev).to_quantized_weight()
    again.load_state_dict(g.state_dict(), assign=True)
    assert torch.equal(again(x, offsets), want)


def test_a_checkpoint_of_another_geometry_is_refused(dev):
    import rtx_b200

    m = rtx_b200.MXFP8LinearEpilogue(256, 128, bias=False, device=dev).to_quantized_weight()
    before = {k: v.clone() for k, v in m.state_dict().items()}
    state = dict(before)
    state["weight_packing_meta"] = before["weight_packing_meta"] + torch.tensor([0, 0, -8, 0])     # K = 248 in the same bytes
    with pytest.raises(RuntimeError, match="K = 248"):
        m.load_state_dict(state)
    assert all(torch.equal(v, before[k]) for k, v in m.state_dict().items())
