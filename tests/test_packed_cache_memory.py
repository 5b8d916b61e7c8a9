"""Caches in four bits: the device memory of closed ones."""
import pytest
import torch

from cake_b200.model import Cache
from tests.test_packed_cache import close_to_rows, ctx_for, rows


@pytest.mark.gpu
def test_closed_caches_give_their_memory_back():
    """A cache of 2.7 GB; up to 1 GiB may stay with the context for the next one."""
    ctx = ctx_for(8, 8, 128, "bf16", max_seq=1 << 17)
    k = rows(16, 3, 8, 128, "bf16", 1)
    free = lambda: torch.cuda.mem_get_info()[0]
    first = Cache(ctx, 16, 16, bits=4)       # (the kernels are loaded with the first calls, and torch takes its first blocks)
    first.write(0, k, k, 0)
    close_to_rows(first.read(0, 0), k, "bf16")
    first.close()
    torch.cuda.synchronize()
    before = free()
    for _ in range(3):
        cache = Cache(ctx, 16, 1 << 17, bits=4)
        cache.write(0, k, k, 0)
        torch.cuda.synchronize()
        assert before - free() > 2.6e9
        close_to_rows(cache.read(0, 0), k, "bf16")
        cache.close()
        assert before - free() < (1 << 30) + (64 << 20)
    small = Cache(ctx, 16, 4096, bits=4)     # 84 MB: of what has stayed, or new
    small.write(0, k, k, 0)
    close_to_rows(small.read(0, 1), k, "bf16")
    ctx.close()
    assert before - free() < 64 << 20
