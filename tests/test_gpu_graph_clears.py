"""Entry points that clear an accumulator first -- the fused silhouette IoU, the deterministic backward, voxelization -- inside a HIP graph:
every replay, with eager work between the replays, equals the eager result on the inputs of that replay, and the graph holds no memset node."""
import ctypes

import numpy as np
import pytest
import torch

import scenes

pytestmark = pytest.mark.gpu


def node_types(graph):
    """hipGraphNodeType of every node of a captured graph (0 kernel, 1 copy, 2 memset)."""
    path = next(l.split()[-1] for l in open('/proc/self/maps') if 'libamdhip64' in l)
    hip = ctypes.CDLL(path)
    raw, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    types = []
    for node in nodes:
        t = ctypes.c_int(-1)
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(t)) == 0
        types.append(t.value)
    return types


def capture(step):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = step()
    types = node_types(graph)
    assert types and 2 not in types, types
    return graph, out


def replays(step, load, check, n=4):
    """`load(i)` writes the inputs of replay i in place; `check(got, want)` compares a replay's outputs with the eager step's."""
    load(0)
    graph, out = capture(step)
    for i in range(n):
        load(i)
        graph.replay()
        got = [t.detach().clone() for t in out]
        torch.cuda.synchronize()
        want = [t.detach().clone() for t in step()]             # eager work between the replays
        torch.cuda.synchronize()
        check(got, want)
        graph.replay()                                          # the same inputs a second time: nothing is left over from the first
        torch.cuda.synchronize()
        check([t.detach().clone() for t in out], want)


def all_equal(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert all(bool(torch.isfinite(b).all()) for b in want)


def test_silhouette_iou_loss_step(native_lib, monkeypatch):
    """One tile per image and the backward pass in a fixed order: no sum depends on the order of atomics, so replays are equal bit for bit."""
    from gendr_amd.functional import silhouette_iou_loss
    monkeypatch.setenv('GENDR_DETERMINISTIC', '1')
    B, isz = 4, 8
    fv = torch.empty(B, 48, 3, 3, device='cuda').requires_grad_(True)
    target = torch.empty(B, isz, isz, device='cuda')

    def load(i):
        with torch.no_grad():
            fv.copy_(torch.from_numpy(scenes.soup(B=B, nf=48, seed=i)[0]))
            target.copy_(torch.from_numpy((np.random.RandomState(i).rand(B, isz, isz) < 0.5).astype(np.float32)))

    def step():
        loss = silhouette_iou_loss(fv, target, image_size=isz, dist_scale=2e-2)
        return loss, torch.autograd.grad(loss, fv)[0]

    replays(step, load, all_equal)


@pytest.mark.parametrize("B,isz", [(2, 64), (1, 200), (3, 512), (1, 512), (1, 1024)])
def test_silhouette_iou_sums(native_lib, B, isz):
    from gendr_amd.functional import silhouette_iou
    fv = torch.empty(B, 48, 3, 3, device='cuda')
    target = torch.empty(B, isz, isz, device='cuda')

    def load(i):
        fv.copy_(torch.from_numpy(scenes.soup(B=B, nf=48, seed=i)[0]))
        target.copy_(torch.from_numpy(np.random.RandomState(i).rand(B, isz, isz).astype(np.float32)))

    # the tiles' sums are added in any order, all terms positive: m additions of relative error 2^-24 each on either side, a tile being
    # cut into eight parts at most; the target's own sum (m = pixels) likewise, and one addition joins the two
    bound = 2 * (8 * ((isz + 7) // 8) ** 2 + isz * isz + 1) * 2.0 ** -24

    def close(got, want):
        for a, b in zip(got, want):
            assert bool(((a - b).abs() <= bound * b.abs()).all()), (a, b)
        assert float(want[0].min()) > 0

    replays(lambda: silhouette_iou(fv, target, image_size=isz, dist_scale=2e-2), load, close)


def test_anti_aliased_iou_loss(native_lib):
    import types
    from gendr_amd import GenDR
    isz = 512
    r = GenDR(image_size=isz, anti_aliasing=True, dist_scale=2e-2)
    mesh = types.SimpleNamespace(face_vertices=torch.empty(1, 48, 3, 3, device='cuda'))
    target = torch.empty(1, isz, isz, device='cuda')

    def load(i):
        mesh.face_vertices.copy_(torch.from_numpy(scenes.soup(B=1, nf=48, seed=i)[0]))
        target.copy_(torch.from_numpy(np.random.RandomState(i).rand(1, isz, isz).astype(np.float32)))

    # two sums of positive terms (m = pixels, as above) on either side, their quotient, at most 1
    bound = 2 * 2 * (isz * isz + 2) * 2.0 ** -24

    def close(got, want):
        assert float((got[0] - want[0]).abs()) <= bound and 0 < float(want[0]) < 1

    replays(lambda: (r.silhouette_iou_loss(mesh, target),), load, close)


def test_deterministic_render(native_lib, monkeypatch):
    from gendr_amd.functional import render
    monkeypatch.setenv('GENDR_DETERMINISTIC', '1')
    B, isz = 2, 64
    fv = torch.empty(B, 48, 3, 3, device='cuda').requires_grad_(True)
    tex = torch.empty(B, 48, 1, 3, device='cuda').requires_grad_(True)
    g = torch.randn(B, 4, isz, isz, device='cuda', generator=torch.Generator('cuda').manual_seed(1))

    def load(i):
        f, t = scenes.soup(B=B, nf=48, seed=i)                  # one of its faces covers the image: it goes through the deferred list
        with torch.no_grad():
            fv.copy_(torch.from_numpy(f))
            tex.copy_(torch.from_numpy(t))

    def step():
        img = render(fv, tex, image_size=isz, dist_func='logistic', dist_scale=2e-2)
        return (img,) + torch.autograd.grad(img, (fv, tex), g)

    replays(step, load, all_equal)


@pytest.mark.parametrize("size", [1, 7, 32, 70])
def test_voxelization(native_lib, size):
    from gendr_amd.functional import voxelization
    faces = torch.empty(2, 20, 3, 3, device='cuda')
    load = lambda i: faces.copy_(torch.from_numpy(np.random.RandomState(i).rand(2, 20, 3, 3).astype(np.float32)))
    replays(lambda: (voxelization(faces, size),), load, all_equal)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("B,size", [(1, 1), (3, 1), (1, 2), (3, 7), (2, 32)])
def test_voxels_at_any_word(native_lib, offset, B, size):
    """The grid is cleared from its first word to its last and nothing beside it is touched, whatever its alignment."""
    n = B * size ** 3
    buf = torch.full((n + 16,), 77, dtype=torch.int32, device='cuda')
    at = buf[4 + offset:4 + offset + n]
    faces = torch.full((B, 1, 9), 0.25, device='cuda')          # one point per item, in voxel (0, 0, 0)
    st = torch.cuda.current_stream().cuda_stream
    e = native_lib.gendr_voxelize(ctypes.c_void_p(faces.data_ptr()), ctypes.c_void_p(at.data_ptr()), None, B, 1, size, ctypes.c_void_p(st))
    assert e == 0
    torch.cuda.synchronize()
    want = torch.zeros(B, size, size, size, dtype=torch.int32)
    want[:, 0, 0, 0] = 1                                        # every other voxel is visible from the border: empty
    assert torch.equal(at.cpu().view(B, size, size, size), want)
    assert bool((buf[:4 + offset] == 77).all()) and bool((buf[4 + offset + n:] == 77).all())
