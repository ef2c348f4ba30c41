"""The serving path over the paged 4-bit cache (esimd_learning_b200/paged.py):
planner, append and attention run together inside the layer stack.  The
attention of every step is compared with float64 attention over what the cache
holds (the append itself is pinned bit for bit in test_kv4.py)."""
import dataclasses

import pytest
import torch

from esimd_learning_b200.chain import SMALL
from oracle import kv4 as K

SHAPE = dataclasses.replace(SMALL, hidden=512, intermediate=1024)


def make(dev, layers=2, num_pages=40, requests=4, max_seq=256, page=16, window=0):
    from esimd_learning_b200.paged import PagedDecoder, PagedKV4Cache, layer_weights
    cache = PagedKV4Cache(layers, SHAPE, num_pages, requests, max_seq, dev, page)
    model = PagedDecoder([layer_weights(SHAPE, seed=i, device=dev) for i in range(layers)], SHAPE, cache, window)
    return model, cache


def hidden(rows, seed, dev):
    return torch.randn(rows, SHAPE.hidden, generator=torch.Generator().manual_seed(seed)).half().to(dev)


def check_last_layer(model, cache, layer):
    last = model.last
    hq, d = SHAPE.num_q_heads, SHAPE.head_dim
    got = last["attention"].cpu()
    ref, vmax = K.attention(last["qkv"][:, :hq].cpu(), cache.pages[layer].cpu(), cache.page_size, cache.scales[layer].cpu(),
                            cache.block_table.cpu(), last["start"].cpu(), cache.context_lens.cpu(), d ** -0.5, model.window)
    # the bound that test_kv4.py derives: output rounding, fp16 probabilities, fp32 scores
    tol = 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2.0 ** -13) * vmax[..., None] + 2.0 ** -25
    assert ((got.double() - ref).abs() <= tol).all()


def test_refuses_unsupported_pages():
    from esimd_learning_b200.paged import PagedKV4Cache
    with pytest.raises(ValueError):
        PagedKV4Cache(1, SHAPE, 4, 1, 64, "cpu", page_size=24)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 20])
def test_prompts_then_tokens(ext, cuda_device, window):
    model, cache = make(cuda_device, window=window)
    lens = [0, 0, 0, 0]
    for step, n in enumerate([[33, 1, 0, 70], [1, 1, 1, 1], [1, 0, 1, 1], [5, 2, 0, 1], [1, 1, 1, 1]]):
        out = model.forward(hidden(sum(n), step, cuda_device), n)
        lens = [a + b for a, b in zip(lens, n)]
        assert cache.context_lens.tolist() == lens and torch.isfinite(out).all()
        check_last_layer(model, cache, 1)
    used = sum(-(-x // 16) for x in lens)
    assert cache.free_count.item() == 40 - used
    rows = [cache.block_table[i, :-(-x // 16)].tolist() for i, x in enumerate(lens)]
    assert len(set(sum(rows, []))) == used  # no page twice


@pytest.mark.gpu
def test_captured_step_equals_eager(ext, cuda_device):
    """Replays advance lengths, pages and slots on the device and give the eager steps' bits."""
    n = [31, 16, 0, 7]
    outs = []
    for captured in (False, True):
        model, cache = make(cuda_device)
        model.forward(hidden(sum(n), 1, cuda_device), n)
        step = model.capture(4) if captured else None
        got = []
        for i in range(20):
            h = hidden(4, 100 + i, cuda_device)
            if captured:
                step.hidden.copy_(h)
                got.append(step.replay().clone())
                junk = [torch.full((64,), -9, dtype=torch.int32, device=cuda_device) for _ in range(50)]  # reuses freed blocks
                del junk
            else:
                got.append(model.forward(h, [1, 1, 1, 1]))
        outs.append((torch.stack(got), cache.context_lens.tolist(), cache.free_count.item(), cache.block_table.clone()))
    assert torch.equal(outs[0][0], outs[1][0]) and outs[0][1:3] == outs[1][1:3] and torch.equal(outs[0][3], outs[1][3])


@pytest.mark.gpu
def test_refusal_and_release(ext, cuda_device):
    """A request without pages is refused whole, its neighbours go on; released pages serve the next one."""
    model, cache = make(cuda_device, num_pages=6)
    a = model.forward(hidden(60, 2, cuda_device), [30, 30, 0, 0])
    out = model.forward(hidden(50, 3, cuda_device), [1, 1, 48, 0])
    assert cache.refused() == [2] and cache.context_lens.tolist() == [31, 31, -1, 0] and cache.free_count.item() == 2
    assert torch.isfinite(out).all() and not model.last["attention"][2:].any()
    check_last_layer(model, cache, 1)
    cache.release(2)
    cache.release(0)
    assert cache.free_count.item() == 4
    again = model.forward(hidden(60, 2, cuda_device)[:30], [30, 0, 0, 0])
    # other row counts take other GEMM tiles, but each row's arithmetic is its own
    torch.testing.assert_close(again, a[:30])


@pytest.mark.gpu
def test_captured_step_keeps_what_it_reads(ext, cuda_device):
    """The step alone is enough: weights and cache live as long as it does."""
    import gc
    import weakref
    model, cache = make(cuda_device, layers=1)
    step = model.capture(2)
    read = [weakref.ref(t) for t in (model.cos_sin, model.layers[0]["qkv"][0], cache.pages, cache.scales, cache.block_table,
                                     cache.context_lens, cache.free_pages, cache.free_count)]
    del model, cache
    gc.collect()
    assert all(r() is not None for r in read)
    step.hidden.copy_(hidden(2, 0, cuda_device))
    assert torch.isfinite(step.replay()).all()


def test_refuses_lengths_without_positions():
    """Positions past the RoPE table would all turn like its last one."""
    from esimd_learning_b200.paged import PagedKV4Cache
    assert PagedKV4Cache(1, SHAPE, 4, 1, SHAPE.max_position, "cpu").block_table.shape == (1, SHAPE.max_position // 64)
    with pytest.raises(ValueError):
        PagedKV4Cache(1, SHAPE, 4, 1, SHAPE.max_position + 1, "cpu")


@pytest.mark.gpu
def test_lengths_up_to_the_last_page(ext, cuda_device):
    """max_seq_len inside a page: the planner hands that page out whole, and attention reads all of it."""
    model, cache = make(cuda_device, num_pages=34, requests=2, max_seq=SHAPE.max_position - 6)
    for step, n in enumerate([[480, 3], [24, 1], [7, 0], [1, 1]]):
        out = model.forward(hidden(sum(n), step, cuda_device), n)
        assert torch.isfinite(out).all()
        check_last_layer(model, cache, 1)
    assert cache.context_lens.tolist() == [512, 5]
    assert cache.max_seq_len == 512 and model.cos_sin.shape[0] >= 512
    model.forward(hidden(1, 9, cuda_device), [1, 0])
    assert cache.refused() == [0]
