"""Voxelization of faces in any memory layout: the native call reads a dense [B, nf, 9] array."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LAYOUTS = {
    'transposed': lambda f: f.transpose(2, 3).contiguous().transpose(2, 3),
    'faces first': lambda f: f.transpose(0, 1).contiguous().transpose(0, 1),
    'every second face': lambda f: f.repeat_interleave(2, dim=1)[:, ::2],
    'one mesh expanded': lambda f: f[:1].expand_as(f),
    'float64': lambda f: f.double().transpose(2, 3).contiguous().transpose(2, 3),
}


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("normalize", [False, True])
def test_layouts(native_lib, layout, normalize):
    from gendr_amd.functional import voxelization
    f = torch.rand(3, 17, 3, 3, device='cuda', generator=torch.Generator('cuda').manual_seed(2))
    if normalize:
        f = f * 20
    view = LAYOUTS[layout](f)
    before = view.clone()
    want = voxelization(view.to(torch.float32).contiguous(), 20, normalize)
    assert torch.equal(voxelization(view, 20, normalize), want) and int(want.sum()) > 0
    assert torch.equal(view, before)                            # the caller's faces are left as they were
