"""flash_attn_tree_with_kvcache on each of its kernels: windows, caps and splits where pages are no multiple of 8 tokens or the
general kernels are asked for, and rows in front of every window that hold NaN or infinities."""
import contextlib

import pytest
import torch

import fa_b200_capi as capi
from tests.test_tree_attention_gpu import check, make

pytestmark = pytest.mark.gpu

KERNELS = [  # head dim, cap, page, policy, the kernel that runs
    (128, 0.0, 64, 0, "sm100_tcgen05_tree"),
    (64, 0.0, 0, 0, "sm100_tcgen05_tree"),
    (64, 20.0, 64, 0, "sm100_tcgen05_2q"),
    (256, 0.0, 16, 0, "sm100_tcgen05_wide"),
    (192, 5.0, 0, 0, "sm100_tcgen05_wide"),
    (128, 0.0, 36, 0, "generic_mma"),
    (64, 20.0, 12, 0, "generic_mma"),
    (256, 0.0, 1, 0, "generic_mma"),
    (96, 5.0, 64, 1, "generic_mma"),
    (40, 0.0, 0, 1, "generic_mma"),
]
IDS = ["-".join(map(str, k)) for k in KERNELS]


@contextlib.contextmanager
def policy(n):
    capi.lib.fa_set_kernel_policy(n)
    try:
        yield
    finally:
        capi.lib.fa_set_kernel_policy(0)


def poison_in_front(c, left, value):
    """Rows of K and V that lie in front of the window of every token."""
    for b, n in enumerate(c["lens"].tolist()):
        for j in range(max(0, n - left)):
            at = (int(c["table"][b, j // c["kc"].shape[1]]), j % c["kc"].shape[1]) if c["table"] is not None else (b, j)
            c["kc"][at] = c["vc"][at] = value


@pytest.mark.parametrize("kernel", KERNELS, ids=IDS)
@pytest.mark.parametrize("left", [0, 37, 130])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_in_front_of_every_window(kernel, left, value):
    d, cap, page, pol, name = kernel
    c = make(torch.bfloat16, d, 6, 2, [300, 77, 500], 9, page, seed=d + page, ragged=True)
    poison_in_front(c, left, value)
    with policy(pol):
        check(c, left=left, softcap=cap)
        assert capi.last_kernel() == name


@pytest.mark.parametrize("kernel", KERNELS, ids=IDS)
@pytest.mark.parametrize("left,num_splits", [(-1, 0), (-1, 2), (-1, 7), (37, 3), (600, 2), (0, 1)])
def test_windows_and_splits(kernel, left, num_splits):
    d, cap, page, pol, name = kernel
    c = make(torch.float16, d, 8, 2, [1500, 3, 700], 21, page, seed=d + page + 1, ragged=True)
    with policy(pol):
        check(c, left=left, softcap=cap, num_splits=num_splits)
        assert capi.last_kernel() == name
