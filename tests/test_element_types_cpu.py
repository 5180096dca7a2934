"""CPU: image operators refuse the element types that only the row operators take (64-bit indices, bfloat16) as any other error."""
import numpy as np
import pytest
import torch


@pytest.fixture()
def host_memory(pkg, monkeypatch):
    """Host tensors pass for device memory: the calls below end before anything is launched."""
    monkeypatch.setattr(pkg.ops, "_device_accessible", lambda t: True)
    monkeypatch.setattr(pkg.cvcuda, "_ingest", lambda t: t._t if isinstance(t, pkg.cvcuda.Tensor) else t)
    monkeypatch.setattr(pkg.cvcuda, "_device", lambda: torch.device("cpu"))
    return pkg


def test_only_tensors_hold_indices(host_memory):
    cv = host_memory.cvcuda
    assert cv.Tensor((2, 3), cv.Type.S64, "NW").dtype == np.int64
    for kind in (np.int64, np.float64, "not a type"):
        with pytest.raises(host_memory.ops.Error) as e:
            cv._torch_dtype(kind)
        assert e.value.status == host_memory.ops.Status.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("kind", [torch.int64, torch.bfloat16])
def test_image_operators_refuse_them(host_memory, kind):
    cv, Error, Status = host_memory.cvcuda, host_memory.ops.Error, host_memory.ops.Status
    x = cv.Tensor((1, 16, 16, 3), kind, "NHWC")
    dst = cv.Tensor((1, 8, 8, 3), np.uint8, "NHWC")
    images = host_memory.ops.ImageBatchVarShape()
    images._images, images._table, images._max_size = [x._t[0]], torch.zeros(1), (16, 16)
    for call in (lambda: cv.resize_crop_convert_reformat_into(dst, x, (8, 8), cv.Interp.LINEAR, (0, 0)),
                 lambda: host_memory.ops._source_of(images), lambda: host_memory.ops._source_of(x._t),
                 lambda: host_memory.ops._dest_of(x._t, "NHWC")):
        with pytest.raises(Error) as e:
            call()
        assert e.value.status == Status.ERROR_INVALID_ARGUMENT


def test_the_allocating_call_refuses_them(host_memory):
    cv, Error = host_memory.cvcuda, host_memory.ops.Error
    for kind in (np.int64, cv.Type.S64):
        with pytest.raises(Error) as e:
            cv.crop_flip_normalize_reformat(None, (1, 8, 8, 3), kind, "NHWC", None, None, None, None)
        assert e.value.status == host_memory.ops.Status.ERROR_INVALID_ARGUMENT
