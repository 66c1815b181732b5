"""Random calls of flash_attn_tree_with_kvcache against the plain form: head dims, groups, trees with holes, lengths, layouts, pages
that are missing, windows with NaN in front of them, caps, splits, tables of angles in both types, and the general kernels."""
import random

import pytest
import torch

from tests.test_tree_attention_gpu import check, make
from tests.test_tree_masks_gpu import policy

pytestmark = pytest.mark.gpu


def draw(seed):
    rng = random.Random(seed)
    hkv = rng.choice([1, 1, 2, 3, 4])
    g = rng.choice([x for x in (1, 2, 3, 4, 5, 7, 8, 12, 16, 32) if x * hkv <= 32])
    d = rng.choice([8, 16, 40, 64, 64, 72, 96, 128, 128, 136, 192, 200, 256])
    t = rng.choice([1, 2, 9, 31, 32, 33, 64, 65, 200, 256]) if rng.random() < 0.4 else rng.randint(1, 40)
    page = rng.choice([0, 0, 1, 8, 12, 16, 24, 36, 40, 48, 64, 64, 96, 128, 256])
    b, hi = rng.randint(1, 5), rng.choice([3, 50, 130, 300, 700, 1500])
    if t * g * hkv * b * hi > 1_500_000:
        hi = 40
    lens = [rng.choice([0, 1, 127, 128, rng.randint(0, hi), rng.randint(0, hi)]) for _ in range(b)]
    rotary = rng.choice([None, None, "half", "interleaved", "partial"]) if d >= 16 else None
    c = make(rng.choice([torch.bfloat16, torch.float16]), d, hkv * g, hkv, lens, t, page, seed, holes=rng.choice([0, 0, 0.2]),
             ragged=rng.random() < 0.4, rotary=rotary, axes=rng.choice([1, 1, 2, 3]) if rotary else 1, extra_pages=rng.randint(0, 3))
    if rotary and rng.random() < 0.4:
        ang = torch.rand(c["cos"].shape, generator=torch.Generator().manual_seed(seed)) * 6.28
        c["cos"], c["sin"] = ang.cos(), ang.sin()
    if page and rng.random() < 0.2:                              # a capacity that ends inside the draft, and lengths past it
        c["table"] = c["table"][:, :max(1, c["table"].shape[1] - 2)].contiguous()
        c["lens"] = c["lens"].clamp(max=c["table"].shape[1] * page + 3)
    if page and rng.random() < 0.15:
        c["table"][rng.randrange(b), rng.randrange(c["table"].shape[1])] = rng.choice([-1, c["kc"].shape[0], 10 ** 9, -2 ** 31])
    left = rng.choice([-1, -1, 0, 1, rng.randint(0, 200)])
    if left >= 0 and rng.random() < 0.6:
        for i, n in enumerate(c["lens"].tolist()):
            for j in range(max(0, min(n, (page or c["kc"].shape[1]) * (c["table"].shape[1] if page else 1)) - left)):
                at = (int(c["table"][i, j // page]), j % page) if page else (i, j)
                if 0 <= at[0] < c["kc"].shape[0]:
                    c["kc"][at] = c["vc"][at] = rng.choice([float("nan"), float("inf")])
    kw = dict(left=left, softcap=rng.choice([0.0, 0.0, 5.0, 30.0]), num_splits=rng.choice([0, 0, 1, 2, 5, 300]))
    return c, kw, int(rng.random() < 0.2)


@pytest.mark.parametrize("block", range(8))
def test_random_calls(block):
    for seed in range(1000 + 40 * block, 1040 + 40 * block):
        c, kw, general = draw(seed)
        with policy(general):
            try:
                check(c, **kw)
            except AssertionError as e:
                raise AssertionError(f"seed {seed}, {kw}: {e}") from e
