"""The forward kernel's pair hints on tiles with many batches of 64 pairs: every batch's slot is written, whatever its place in the tile."""
import numpy as np
import pytest

import parity

pytestmark = pytest.mark.gpu


def big_faces(B, nf, seed=0):
    """Faces that each cover much of the image: with 2 x 2 tiles of 64 pixels a tile lists thousands of pairs."""
    rs = np.random.RandomState(seed)
    fv = np.zeros((B, nf, 3, 3), np.float32)
    fv[..., :2] = rs.uniform(-1.2, 1.2, (B, nf, 3, 2))
    fv[..., 2] = rs.uniform(1.5, 5.0, (B, nf, 3))
    return fv, rs.uniform(0, 1, (B, nf, 1, 3)).astype(np.float32)


@pytest.mark.parametrize("team", [-1, 1])
@pytest.mark.parametrize("rgb", ['softmax', 'hard'])
@pytest.mark.parametrize("B,nf", [(1, 17), (2, 300)])
def test_hints_of_every_batch_arrive(oracle_mod, native_lib, team, rgb, B, nf):
    isz = 16
    fv, tex = big_faces(B, nf, seed=nf)
    opts = dict(dist_scale=1e-2, aggr_rgb_func=rgb, team=team)
    grad = np.random.RandomState(1).randn(B, 4, isz, isz).astype(np.float32)
    o = parity.run_oracle(fv, tex, isz, dict(opts, team=0), grad)
    on = parity.run_hip(fv, tex, isz, dict(opts, pair_hints=1), grad)
    off = parity.run_hip(fv, tex, isz, dict(opts, pair_hints=-1), grad)
    assert np.array_equal(on['rgba'], off['rgba']) and np.array_equal(on['aggrs_info'], off['aggrs_info'])
    # the two calls add the same partials in another order: a sum of n terms is within n eps / 2 of the exact one relative to the sum of
    # the magnitudes, n <= 256 pixels a face, for either call
    bound = 2 * 256 * 2.0 ** -24
    for k, ak in (('grad_faces', 'abs_faces'), ('grad_textures', 'abs_textures')):
        scale = np.maximum(o[ak].reshape(on[k].shape), 1e-30)
        err = np.abs(on[k].astype(np.float64) - off[k]) / scale
        assert err.max() <= bound, (k, float(err.max()))
        assert np.abs(off[k]).max() > 0
