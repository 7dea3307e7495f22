"""The MXFP4 and routing calls go to torch's current stream, with and without
torch's private shortcut to its handle."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shortcut", [True, False])
def test_calls_go_to_the_current_stream(monkeypatch, shortcut):
    import torch

    import minirun_hip as M

    if not shortcut:
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    x = torch.randn(5, 64, device="cuda")
    w = M.mxfp4_quantize(torch.randn(16, 64, device="cuda"))
    want = M.mxfp4_mm(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert M._call_stream(x.device, None)[0] == s.cuda_stream
        got = M.mxfp4_mm(x, w)
    s.synchronize()
    assert torch.equal(got, want)
    assert M._call_stream(x.device, None)[0] == torch.cuda.current_stream().cuda_stream
