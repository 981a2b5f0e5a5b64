"""The training operators' kernels against float64 at the sizes by which a launch takes
another form: workgroups that take several windows, four waves where there are workgroups
enough, tiles of 128.  A card of 256 compute units is assumed only for which form is met:
the results have to hold on any.  Tolerances as in ``test_gpu_training_ops``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import frame_analytics_amd as fa
from oracle import training as ref
from tests.test_gpu_training_ops import DT, ORTHO, POLAR, STEEP, check_attention, near

pytestmark = pytest.mark.gpu


def window_mask(gen, m, heads, n):
    """Half of the pairs; a query that sees nothing, a key that nothing sees, and (of
    three entries or more) an entry that sees nothing."""
    mask = torch.rand(m, heads, n, n, generator=gen) < 0.5
    mask[0, :, 3 % n] = False
    mask[-1, :, :, n // 2] = False
    if m > 2:
        mask[1] = False
    return mask


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("h,w,d", [(8, 8, 32), (7, 7, 30), (4, 6, 33), (8, 8, 64)])
@pytest.mark.parametrize("heads", [1, 2])
def test_masks_in_windows(gpu, dt, h, w, d, heads):
    """A mask for all heads or for each, more windows than entries of it."""
    n = h * w
    mask = window_mask(torch.Generator().manual_seed(n), 3, heads, n)
    check_attention(dt, 9, 2, 2, n, n, d, fa.GridPositions(h, w), ref.grid_rows(h, w),
                    mask=mask.cuda())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("h,w", [(8, 8), (5, 7), (10, 11), (16, 16)])
def test_key_lengths_in_windows(gpu, dt, h, w):
    n = h * w
    lens = torch.tensor([n, 0, 1, n - 1, n // 2, 2 * n, 33 % n], dtype=torch.int64).cuda()
    check_attention(dt, 7, 2, 2, n, n, 32, fa.GridPositions(h, w), ref.grid_rows(h, w),
                    key_lengths=lens)


@pytest.mark.parametrize("dt", list(DT))
def test_causal_windows(gpu, dt):
    check_attention(dt, 3, 2, 2, 64, 64, 32, fa.GridPositions(8, 8), ref.grid_rows(8, 8), causal=True)
    check_attention(dt, 3, 2, 2, 132, 132, 32, fa.GridPositions(11, 12), ref.grid_rows(11, 12),
                    causal=True)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("h,w,d,masked", [(8, 8, 32, True), (7, 7, 30, True), (8, 8, 30, False),
                                          (4, 4, 16, True)])
def test_many_windows_for_each_workgroup(gpu, dt, h, w, d, masked):
    """Workgroups that walk over windows: 1031 of 4 heads are four or five each, with
    masks that repeat over 64 and key lengths of every kind."""
    b, heads, n = 1031, 4, h * w
    gen = torch.Generator().manual_seed(n + d)
    kw = {"key_lengths": torch.randint(0, n + 5, (b,), generator=gen).cuda()}
    if masked:  # 1031 is a prime: as many masks as windows
        kw["mask"] = window_mask(gen, b, 1, n).cuda()
    check_attention(dt, b, heads, heads, n, n, d, fa.GridPositions(h, w), ref.grid_rows(h, w), **kw)


@pytest.mark.parametrize("dt", list(DT))
def test_many_windows_with_a_repeating_mask(gpu, dt):
    gen = torch.Generator().manual_seed(7)
    check_attention(dt, 1036, 2, 2, 64, 64, 32, fa.GridPositions(8, 8), ref.grid_rows(8, 8),
                    mask=window_mask(gen, 7, 1, 64).cuda())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("h,w,b", [(10, 11, 301), (12, 12, 130), (16, 16, 66)])
def test_many_wide_windows(gpu, dt, h, w, b):
    """Sums by pair that stay in registers over several windows."""
    n = h * w
    check_attention(dt, b, 4, 4, n, n, 32, fa.GridPositions(h, w), ref.grid_rows(h, w), seed=b)


@pytest.mark.parametrize("dt", list(DT))
def test_wide_windows_with_masks(gpu, dt):
    gen = torch.Generator().manual_seed(9)
    check_attention(dt, 6, 2, 2, 110, 110, 30, fa.GridPositions(10, 11), ref.grid_rows(10, 11),
                    mask=window_mask(gen, 3, 2, 110).cuda())
    check_attention(dt, 4, 4, 2, 300, 300, 48, fa.GridPositions(15, 20), ref.grid_rows(15, 20),
                    mask=window_mask(gen, 2, 1, 300).cuda())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("heads,hk", [(2, 2), (4, 2)])
def test_one_element_at_a_time(gpu, dt, heads, hk):
    """Views with an odd offset and an odd dimension, gradients included."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    for pos, n, d in ((fa.GridPositions(7, 8), 56, 29), (fa.GridPositions(9, 9), 81, 31),
                      (fa.LinePositions(8, 20), 150, 45)):
        wide = torch.randn(3, n, heads + 2 * hk, d + 2, generator=gen, device="cuda").to(DT[dt])
        cut = wide[..., 1:d + 1].transpose(1, 2)
        ts = [cut[:, :heads], cut[:, heads:heads + hk], cut[:, heads + hk:]]
        table = torch.randn(pos.rows, heads, generator=gen, device="cuda").to(DT[dt])
        g = torch.randn(3, n, heads, d + 2, generator=gen, device="cuda").to(DT[dt])[..., 1:d + 1]
        plain = [t.contiguous().requires_grad_(True) for t in ts]
        want = fa.relative_attention(*plain, table, pos)
        want.backward(g.transpose(1, 2).contiguous())
        ts = [t.detach().requires_grad_(True) for t in ts]
        got = fa.relative_attention(*ts, table, pos)
        got.backward(g.transpose(1, 2))
        assert torch.equal(got, want)
        assert all(torch.equal(x.grad, y.grad) for x, y in zip(ts, plain))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("b,h,hk,lk,d", [(1, 4, 1, 240, 64), (1, 8, 2, 960, 128), (1, 1, 1, 129, 30),
                                         (2, 2, 2, 5000, 64)])
def test_a_new_token_of_one_or_two_sequences(gpu, dt, b, h, hk, lk, d):
    lens = torch.tensor([lk - 3, lk][:b], dtype=torch.int32)
    start = lens - 1
    pos = fa.LinePositions(32, 128, bidirectional=False)
    rows = np.stack([ref.line_rows(1, lk, int(s), 32, 128, False) for s in start])
    check_attention(dt, b, h, hk, 1, lk, d, pos, rows, key_lengths=lens.cuda(),
                    q_start=start.cuda())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("lq,h,hk", [(2, 8, 1), (5, 4, 2), (16, 4, 4), (16, 8, 4), (33, 4, 4)])
def test_few_queries_against_a_ragged_cache(gpu, dt, lq, h, hk):
    """Several new tokens of each sequence, their own starts, causal, and a mask."""
    b, lk, d = 3, 1111, 40
    lens = torch.tensor([lk, 400, lq])
    start = lens - lq
    pos = fa.LinePositions(16, 40)
    rows = np.stack([ref.line_rows(lq, lk, int(s), 16, 40) for s in start])
    kw = {"causal": True, "key_lengths": lens.cuda(), "q_start": start.cuda()}
    check_attention(dt, b, h, hk, lq, lk, d, pos, rows, **kw)
    gen = torch.Generator().manual_seed(lq)
    mask = torch.rand(3, h, lq, lk, generator=gen) < 0.5
    mask[1, :, 0] = False
    check_attention(dt, b, h, hk, lq, lk, d, pos, rows, mask=mask.cuda(), **kw)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("b,h,hk,n,d,causal", [
    (16, 16, 16, 140, 64, True),   # four waves, one group of them
    (8, 16, 16, 135, 64, False),   # four waves in two groups
    (8, 16, 16, 160, 20, True),
    (8, 16, 4, 131, 128, True),    # heads of 128, shared
    (8, 16, 2, 150, 64, True),     # and their key heads' workgroups few
    (40, 8, 8, 60, 40, False)])
def test_lines_of_many_workgroups(gpu, dt, b, h, hk, n, d, causal):
    pos = fa.LinePositions(16, 40, bidirectional=not causal)
    rows = ref.line_rows(n, n + 3, 3, 16, 40, not causal)
    check_attention(dt, b, h, hk, n, n + 3, d, pos, rows, causal=causal, q_start=3)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("batch,m,n", [
    (128, 200, 250),   # tiles of 128 in every product
    (12, 500, 1400),   # tiles of 128 in the last, of 64 in the symmetric ones
    (30, 250, 230),    # tiles of 64, one group of waves in every product
    (20, 130, 640),    # one group in the last, four in the symmetric ones
    (600, 70, 65),
    (600, 40, 130)])  # of up to 64 rows: tiles of 64 however many
def test_updates_of_many_tiles(gpu, dt, batch, m, n):
    gen = torch.Generator().manual_seed(m)
    g = (1e-3 * torch.randn(batch, m, n, generator=gen)).to(DT[dt])
    for steps, coefficients in ((5, STEEP), (2, POLAR)):
        got = fa.orthogonalize(g.cuda(), steps=steps, coefficients=coefficients)
        for i in (0, 1, batch // 2, batch - 1):
            want = ref.orthogonalize(g[i].double().numpy(), steps, coefficients)
            near(got[i], want, ORTHO[dt], i)
        again = fa.orthogonalize(g.cuda(), steps=steps, coefficients=coefficients)
        assert torch.equal(got, again)


@pytest.mark.parametrize("dt", list(DT))
def test_an_update_does_not_depend_on_its_neighbours(gpu, dt):
    gen = torch.Generator().manual_seed(1)
    g = torch.randn(140, 200, 250, generator=gen).to(DT[dt]).cuda()
    got = fa.orthogonalize(g)
    g[:70] = float("nan")
    again = fa.orthogonalize(g)
    assert torch.equal(got[70:], again[70:]) and torch.isnan(again[:70]).all()
