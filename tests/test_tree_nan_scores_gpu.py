"""NaN in a query or in a K row that is seen reaches the output and the LSE of the rows it belongs to, and no others: whichever
kernel runs, wherever the key is in its tile, and wherever the list of keys is cut."""
import math

import pytest
import torch

import fa_b200_capi as capi
from tests.test_tree_attention_gpu import call, make
from tests.test_tree_masks_gpu import IDS, KERNELS, policy
from tests.tree_reference import out_bound, tree_attention

pytestmark = pytest.mark.gpu


def check(c, left=-1, softcap=0.0, num_splits=0):
    out, lse, _, _ = call(c, left, softcap, num_splits)
    ro, rl, mag = tree_attention(c["q"], c["kc"].clone(), c["vc"].clone(), c["k"], c["v"], c["parents"], c["lens"], c["table"], left=left, softcap=softcap)
    bad = ro.isnan()
    assert bad.any() and not bad.all()
    assert torch.equal(out.isnan(), bad)
    assert ((out.double() - ro).abs()[~bad] <= out_bound(ro, mag, out.dtype)[~bad]).all()
    assert torch.equal(lse.isnan(), rl.isnan())
    fin = torch.isfinite(rl)
    assert torch.equal(lse.isinf(), rl.isinf())
    assert ((lse.double() - rl)[fin].abs() <= 4e-5 * rl[fin].abs().clamp_min(1)).all()


def place(c, b, j):
    page = c["kc"].shape[1]
    return (int(c["table"][b, j // page]), j % page) if c["table"] is not None else (b, j)


@pytest.mark.parametrize("kernel", KERNELS, ids=IDS)
@pytest.mark.parametrize("num_splits", [0, 1, 4])
def test_nan_in_a_query(kernel, num_splits):
    d, cap, page, pol, name = kernel
    c = make(torch.bfloat16, d, 6, 2, [1500, 77, 900], 9, page, seed=d + page + 2, ragged=True)
    c["parents"][:, 4] = -1
    c["q"][0, 4, 1, d // 2] = math.nan
    c["q"][2, 4, 5] = math.nan
    c["parents"][1, 8], c["q"][1, 8] = -2, math.nan             # no token: zeros and +inf all the same
    with policy(pol):
        check(c, softcap=cap, num_splits=num_splits)
        assert capi.last_kernel() == name


@pytest.mark.parametrize("kernel", KERNELS, ids=IDS)
@pytest.mark.parametrize("num_splits", [0, 1, 4])
@pytest.mark.parametrize("left", [-1, 300])
def test_nan_in_a_key(kernel, num_splits, left):
    """One row in each sequence, at an even and an odd place of a group of 16 keys, in tiles that all tokens see in full and in
    the last one; with a window some tokens do not see them."""
    d, cap, page, pol, name = kernel
    c = make(torch.float16, d, 6, 2, [1500, 1301, 900, 130], 9, page, seed=d + page + 3)
    for b, j in enumerate((1296, 1011, 600, 129)):
        c["kc"][place(c, b, j)][b % 2, d - 1] = math.nan
    with policy(pol):
        check(c, left=left, softcap=cap, num_splits=num_splits)
        assert capi.last_kernel() == name


@pytest.mark.parametrize("hq,hkv,t,lens,where", [
    (8, 1, 16, [20000], 9000), (2, 2, 3, [12000], 5000), (32, 1, 20, [3000, 1, 40], 1700), (4, 4, 40, [2000] * 9, 1000)])
@pytest.mark.parametrize("j", [0, 1, 6, 15, 64])
def test_a_key_in_the_middle_of_a_cut_sequence(hq, hkv, t, lens, where, j):
    c = make(torch.bfloat16, 64, hq, hkv, lens, t, 64, seed=t + len(lens))
    c["kc"][place(c, 0, where // 128 * 128 + j)][0, 3] = math.nan
    if hkv == 1 and len(lens) == 1:                             # leave rows that are not NaN
        c["parents"][0, -1] = -2
    check(c)
    assert capi.last_kernel() == "sm100_tcgen05_tree"


@pytest.mark.parametrize("num_splits", [0, 1])
def test_a_draft_token_whose_key_is_nan(num_splits):
    """Its descendants are NaN, its siblings are not."""
    c = make(torch.bfloat16, 128, 8, 2, [700, 30], 10, 64, seed=5)
    c["parents"] = torch.tensor([[-1, 0, 0, 1, 2, 3, 4, -1, 7, 8]] * 2, dtype=torch.int32)
    c["k"][:, 1] = math.nan
    check(c, num_splits=num_splits)


@pytest.mark.parametrize("kernel", KERNELS, ids=IDS)
@pytest.mark.parametrize("num_splits", [0, 1, 4])
@pytest.mark.parametrize("j", [0, 1, 5, 64, 127])
def test_infinite_scores(kernel, num_splits, j):
    """A score of +inf makes inf - inf = NaN of its row's softmax, one of -inf has no weight, and the cap makes +-cap of both."""
    d, cap, page, pol, name = kernel
    c = make(torch.bfloat16, d, 6, 2, [1500, 900], 9, page, seed=d + page + 4)
    for b, tile in enumerate((5, 3)):
        row = torch.zeros(2, d)
        row[:, 2] = math.inf
        c["kc"][place(c, b, tile * 128 + j)] = row.bfloat16()
    with policy(pol):
        out, lse, _, _ = call(c, -1, cap, num_splits)
        assert capi.last_kernel() == name
    ro, rl, mag = tree_attention(c["q"], c["kc"].clone(), c["vc"].clone(), c["k"], c["v"], c["parents"], c["lens"], c["table"], softcap=cap)
    bad = (c["q"][..., 2:3] > 0).expand_as(out) & (cap == 0)
    assert torch.equal(ro.isnan(), bad) and torch.equal(out.isnan(), bad)
    assert ((out.double() - ro).abs()[~bad] <= out_bound(ro, mag, out.dtype)[~bad]).all()
    fin = torch.isfinite(rl)
    assert torch.equal(fin, torch.isfinite(lse)) and ((lse.double() - rl)[fin].abs() <= 4e-5 * rl[fin].abs().clamp_min(1)).all()
