"""The cache's memory and streams other than the one it was made on."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["release", "del"])
@pytest.mark.parametrize("current", [False, True])
def test_memory_is_not_handed_out_while_another_stream_works_on_it(pxq, how, current):
    """Released with work under way on a side stream, named in the call or current: torch may give the memory to nobody else
    before that work is done."""
    import torch

    side = torch.cuda.Stream()
    x = torch.ones((70, 128), device="cuda")
    pxq.KVCache(1, 100, 2, 64).append(x, x)  # (a kernel's first launch loads it, which waits for the device)
    cache = pxq.KVCache(1, 100_000, 2, 64)
    with torch.cuda.stream(side):
        torch.cuda._sleep(1000)
    at, size = cache.memory.data_ptr(), cache.memory.numel()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(500_000_000)
        if current:
            cache.append(x, x)
    if not current:
        cache.append(x, x, stream=side)
    if how == "release":
        cache.release()
    else:
        del cache
    assert not side.query()
    other = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert other.data_ptr() != at
    side.synchronize()
    pxq.synchronize()
