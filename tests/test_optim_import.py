"""compressor_b200.optim under a torch that was built without CUDA: it can be
imported, and its checks of lists refuse what they refuse anywhere."""
import importlib.util

import pytest

torch = pytest.importorskip("torch")


def test_import_without_cuda_in_torch(monkeypatch):
    from compressor_b200 import optim as whole
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    spec = importlib.util.spec_from_file_location("compressor_b200.optim_without_cuda", whole.__file__)
    optim = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(optim)
    with pytest.raises(ValueError, match="CUDA device is wanted"):
        optim.GradNorm([torch.zeros(3)])
    with pytest.raises(TypeError):
        optim.AdamW([1.0], [torch.zeros(3)])
