"""clip_grad_norm_, no GPU: strided gradients that share memory are refused, those that only interleave pass
on (to the refusal of CPU tensors)."""

import random

import pytest
import torch

import lewm_flash_b200 as lf

BASE = torch.zeros(40, 60)
G = torch.zeros(30, 30)


def clip(*grads):
    params = []
    for g in grads:
        params.append(torch.nn.Parameter(torch.empty_like(g)))
        params[-1].grad = g
    lf.clip_grad_norm_(params, 1.0)


@pytest.mark.parametrize("grads", [
    (G, G.t()),
    (G.t(), G),
    (BASE[:, :20], BASE[:, 19:40]),
    (BASE[:, :20], BASE[3]),
    (BASE[:, 10:20].t(), BASE[5:6, :11]),
    (BASE[::2, ::2], BASE[::2, 2:]),
    (BASE[::2], BASE[4:9, 30:].t()),
    (BASE[:, 5:15], torch.zeros(7), BASE[:, 20:50].t(), BASE[2, 49:52]),
    (BASE[:, 5], BASE[:, 5].clone()[:3], BASE[39, 5:6]),
    (BASE.view(-1)[::3], BASE.view(-1)[::7]),
    (BASE[:, :2], BASE.view(torch.float16)[:, 3:5]),  # of two types on the same bytes
])
def test_gradients_that_share_memory_are_refused(grads):
    with pytest.raises(ValueError, match="overlap in memory"):
        clip(*grads)


@pytest.mark.parametrize("grad", [BASE[0, :1].expand(3), BASE.as_strided((5, 3), (2, 1)), BASE[:, :1].expand(40, 4),
                                  BASE.as_strided((4, 3, 2), (60, 1, 2))])
def test_gradients_that_share_memory_with_themselves_are_refused(grad):
    with pytest.raises(ValueError, match="shares memory between its own elements"):
        clip(torch.zeros(3), grad)


@pytest.mark.parametrize("grads", [
    (BASE[:, :20], BASE[:, 20:40], BASE[:, 40:].t()),
    (BASE[:, 5:15], BASE[3, 20:50], BASE[:, :5], BASE[4:, 15:20]),
    (BASE[::2, ::2], BASE[::2, 1::2], BASE[1::2, ::2], BASE[1::2, 1::2].t()),
    (BASE.view(-1)[::3], BASE.view(-1)[1::3], BASE.view(-1)[2::6]),
    (BASE[::2], BASE[1::2]),
    (BASE[:0, 1:], BASE[:, 1:], BASE[:0, 3:].t()),
    (BASE[:20, 30:], BASE[20:, 30:], BASE[:, :30]),
    (BASE[::2, ::2],),
    (G.t(), torch.zeros(4, 1).expand(4, 1), torch.zeros(6, 2)[:, 0]),
])
def test_gradients_that_only_interleave_are_taken(grads):
    with pytest.raises(ValueError, match="need a CUDA device"):
        clip(*grads)


def test_interleaved_quarters_of_a_large_buffer_are_taken():
    big = torch.zeros(3000, 3000)
    with pytest.raises(ValueError, match="need a CUDA device"):
        clip(*[big[i::2, j::2] for i in (0, 1) for j in (0, 1)])


@pytest.mark.parametrize("seed", range(40))
def test_refused_exactly_where_elements_meet(seed):
    """Random nested views of one buffer against the sets of their elements."""
    r = random.Random(seed)
    buf = torch.zeros(4000)

    def view():
        sizes, strides, span = [], [], 1
        for _ in range(r.randint(1, 3)):
            sizes.append(r.randint(1, 5))
            strides.append(span + r.randint(0, 6))
            span += (sizes[-1] - 1) * strides[-1]
        order = list(range(len(sizes)))
        r.shuffle(order)
        return buf.as_strided([sizes[i] for i in order], [strides[i] for i in order], r.randint(0, 300))

    places = torch.arange(4000)
    for _ in range(100):
        views = [view() for _ in range(r.randint(2, 4))] + [buf[3000::2]]  # one strided at least
        seen = torch.cat([places.as_strided(v.shape, v.stride(), v.storage_offset()).reshape(-1) for v in views])
        meets = seen.unique().numel() < seen.numel()
        with pytest.raises(ValueError, match="overlap in memory" if meets else "need a CUDA device"):
            clip(*views)
