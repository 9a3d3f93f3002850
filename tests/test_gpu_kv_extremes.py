"""Attention over values whose scales are at the ends of fp32, against 64 bits.

A probability times such a scale is rounded to bf16, as every probability is; below 2^-126 that is to a multiple of 2^-133, off
by 2^-134 at most.  Relative to the row's largest score the probabilities add up to 1 or more, and the kernels' reference is
never above that score: the rows' outputs are off by at most 2^-134 sum |v8| / sum exp(x - max) more than kv_ref.bound has."""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("scale", [2.0 ** 90, 2.0 ** 61, 2.0 ** -61, 1e-30, 2.0 ** -118, 2.0 ** -126, 1e-38, 2.0 ** -130, 2.0 ** -133])
@pytest.mark.parametrize("steep", [0.0, 0.01])
@pytest.mark.parametrize("rows,blocks", [(1, 5), (1, 64), (20, 64), (200, 5), (200, 24), (200, 64)])
def test_value_scales_at_the_ends_of_fp32(rows, blocks, steep, scale):
    """8-bit values of one sign, so that what is lost shows: outputs are 64 to 127 scales.  All probabilities alike, or within a
    factor of about 2 of each other."""
    import h3mi
    rng = np.random.default_rng(rows + blocks)
    heads, dim = 2, 128
    ref = R.Cache(blocks, heads, dim, seed=rows)
    ref.v[:] = rng.integers(64, 128, ref.v.shape)
    ref.vs[:], ref.ks[:] = scale, steep * 0.01
    tables = rng.permutation(blocks)[None].astype(np.int32)
    end = blocks * 64 - 9
    q = torch.from_numpy(rng.standard_normal((1, rows, heads, dim))).to(torch.bfloat16)
    out = h3mi.kv_attention(q.to(DEV), ref.to(), _i32(tables), _i32([end]), causal=True).double().cpu().numpy()
    x = q.double().numpy()
    want, mag, top = R.attention(ref, x, tables, [end], [rows], True)
    k, v, _ = R.tokens(ref, tables[0], end)
    extra = np.zeros((1, rows, heads, 1))
    for h in range(heads):
        s = x[0, :, h] @ k[:, h].T * dim ** -0.5
        s[np.arange(end) > (end - rows + np.arange(rows))[:, None]] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        extra[0, :, h, 0] = 2.0 ** -134 * 127 * np.isfinite(s).sum(1) / p.sum(1)
    bound = R.bound(want, mag, top, dim) - 1e-30 + extra
    # the result's own rounding, where bf16 is below its normal numbers too
    bound += 2.0 ** -134
    assert (np.abs(out - want) <= bound).all(), (np.abs(out - want) / bound).max()
    assert (bound < 0.6 * np.abs(want)).all() if scale >= 2.0 ** -130 else True  # zeros would not do


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 30.0])
@pytest.mark.parametrize("rows,blocks", [(1, 64), (20, 64), (200, 24), (200, 64)])
def test_scales_of_scores_over_joined_parts(rows, blocks, scale):
    """A scale of 0 is the mean of the values, a negative one turns the scores round, a steep one leaves a token or two."""
    import h3mi
    from h3mi import _lib
    rng = np.random.default_rng(rows * blocks)
    heads, dim = 2, 128
    assert _lib.lib.h3mi_kv_attention_workspace(1, rows, heads, heads, dim, blocks, 0) > 0
    ref = R.Cache(blocks, heads, dim, seed=blocks)
    ref.ks *= 0.2
    ref.ks[3], ref.k[3] = 0, 0
    ref.vs[5], ref.v[5] = 0, 0
    tables = rng.permutation(blocks)[None].astype(np.int32)
    end = blocks * 64 - 9
    q = torch.from_numpy(rng.standard_normal((1, rows, heads, dim))).to(torch.bfloat16)
    out = h3mi.kv_attention(q.to(DEV), ref.to(), _i32(tables), _i32([end]), scale=scale).double().cpu().numpy()
    want, mag, top = R.attention(ref, q.double().numpy(), tables, [end], [rows], False, scale)
    assert (np.abs(out - want) <= R.bound(want, mag, top, dim)).all()
