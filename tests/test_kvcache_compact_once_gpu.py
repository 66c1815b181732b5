"""kvcache_compact moves rows in place: a cache that is given twice would be compacted twice."""
import pytest
import torch

import flash_attn_npu_3 as fa

pytestmark = pytest.mark.gpu


def test_a_cache_given_twice_is_refused():
    stack = torch.randn(3, 6, 16, 2, 64, device="cuda").bfloat16()
    before = stack.clone()
    lens = torch.tensor([5, 40], dtype=torch.int32, device="cuda")
    kept = torch.tensor([[1, 3, 6], [0, 2, 7]], dtype=torch.int32, device="cuda")
    table = torch.arange(6, dtype=torch.int32, device="cuda").reshape(2, 3)
    for caches in ([stack[0], stack[0]], [stack, stack[1]], [stack[2], stack], [stack[0], stack[1], stack[0][..., :32]]):
        with pytest.raises(RuntimeError, match="once"):
            fa.kvcache_compact(caches, lens, kept, page_table=table)
        fa.kvcache_copy_pages(caches, lens[:1], lens[:1])       # where nothing moves in place a list may name one twice
    assert torch.equal(stack, before)
    both = before.clone()
    want = fa.kvcache_compact(both, lens, kept, page_table=table)
    for caches in ([stack[0], stack[1], stack[2]], ):
        assert torch.equal(fa.kvcache_compact(caches, lens, kept, page_table=table), want) and torch.equal(stack, both)
    # halves of one tensor, interleaved in memory, are caches of their own
    stack.copy_(before)
    assert torch.equal(fa.kvcache_compact((x for x in (stack[..., :32], stack[..., 32:])), lens, kept, page_table=table), want) and torch.equal(stack, both)
