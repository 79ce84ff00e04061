"""lb_rotary over slices of one tensor that lie between one another, in place and apart; what lies beside the rows stays.

Each result is compared bit for bit with the same rows turned by themselves (test_gpu_rotary holds those against the definition)."""
import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce

pytestmark = pytest.mark.gpu
B, S, H, K, D = 3, 4, 6, 2, 64


def rotary_of(device, dims=D):
    return lb.Rotary(lb.rotary_frequencies(dims, device=device), pairs='neighbours', scale=0.75)


# Two slices of one buffer as [B, S, heads, D], by how its axes lie.
LAYOUTS = {
    'rows': ((B, S, H + K, D), lambda t: (t[:, :, :H], t[:, :, H:])),
    'rows, keys first': ((B, S, K + 1 + H, D), lambda t: (t[:, :, K + 1:], t[:, :, :K])),
    'heads': ((B, H + K, S, D), lambda t: (t[:, :H].transpose(1, 2), t[:, H:].transpose(1, 2))),
    'pairs of heads': ((B, S, H, 2, D), lambda t: (t[:, :, :, 0], t[:, :, :K, 1])),
    'heads of the batch': ((H + K, B, S, D), lambda t: (t[:H].permute(1, 2, 0, 3), t[H:].permute(1, 2, 0, 3))),
    'blocks of a sequence': ((B, S * (H + K), D), lambda t: (t[:, :S * H].unflatten(1, (S, H)), t[:, S * H:].unflatten(1, (S, K)))),
    'every other sequence': ((2 * B, S, H, D), lambda t: (t[::2], t[1::2, :, :K])),
    'every other row': ((B, 2 * S, H, D), lambda t: (t[:, ::2], t[:, 1::2, 1:K + 1])),
    'halves of a row': ((B, S, H, 2 * D), lambda t: (t[..., :D], t[:, :, :K, D:])),
    'padded sequences': ((B, S * (H + K) * D + 40), lambda t: tuple(
        t.as_strided((B, S, n, D), (t.stride(0), (H + K) * D, D, 1), at) for n, at in ((H, 0), (K, H * D)))),
}


@pytest.mark.parametrize('name', LAYOUTS)
@pytest.mark.parametrize('type', [torch.float16, torch.float32])
def test_slices_of_one_tensor(device, name, type):
    announce('rotary layouts', name, type)
    shape, cut = LAYOUTS[name]
    whole = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(type).to(device)
    rotary, position = rotary_of(device), torch.tensor([5, 0, 1000], device=device)
    q, k = (t.clone() for t in cut(whole))
    want = lb.rotary(q, position, rotary), lb.rotary(k, position, rotary)
    expected = whole.clone()
    for slot, value in zip(cut(expected), want):
        slot.copy_(value)
    apart = whole.clone()
    out, out_k = cut(apart)
    assert lb.rotary(q, position, rotary, k=k, out=out, out_k=out_k)[0] is out
    assert torch.equal(apart, expected)
    q, k = cut(whole)
    lb.rotary(q, position, rotary, k=k, out=q, out_k=k)
    assert torch.equal(whole, expected)


def test_into_the_other_half(device):
    """From one slice of a tensor into another that lies between its rows."""
    announce('rotary other half')
    whole = torch.randn((B, S, 2, H, D), generator=torch.Generator().manual_seed(2)).half().to(device)
    before, rotary, position = whole.clone(), rotary_of(device), torch.tensor([1, 2, 3], device=device)
    lb.rotary(whole[:, :, 1], position, rotary, out=whole[:, :, 0])
    assert torch.equal(whole[:, :, 1], before[:, :, 1])
    assert torch.equal(whole[:, :, 0], lb.rotary(before[:, :, 1].contiguous(), position, rotary))


def test_only_rows_apart_are_taken(device):
    """Slices with any strides of a small buffer: a call is taken only where no row of one is a row of the other."""
    announce('rotary any strides')
    rng, dim, taken, refused = np.random.default_rng(3), 4, 0, 0
    rotary = rotary_of(device, dim)
    for _ in range(400):
        b, s, h, kh = (int(n) for n in rng.integers(1, 4, 4))
        unit = [int(x) for x in rng.choice([4, 8, 12, 16, 24, 32, 48, 64, 96], 3)]
        strides = [unit, unit if rng.random() < 0.8 else [int(x) for x in rng.choice([4, 8, 16, 32, 64], 3)]]
        places = [0, int(rng.choice([4, 8, 12, 16, 32, 64, 2, 100]))]
        base = torch.randn(1200, generator=torch.Generator().manual_seed(4)).half().to(device)
        q, k = (base.as_strided((b, s, n, dim), (*st, 1), at) for n, st, at in zip((h, kh), strides, places))
        at = torch.arange(1200)
        sets = [at.as_strided(t.shape, t.stride(), t.storage_offset()).reshape(-1).tolist() for t in (q, k)]
        each = all(len(set(x)) == len(x) for x in sets)
        apart = each and not set(sets[0]) & set(sets[1])
        position = torch.arange(b, device=device)
        want = lb.rotary(q.clone(), position, rotary), lb.rotary(k.clone(), position, rotary)
        try:
            lb.rotary(q, position, rotary, k=k, out=q, out_k=k)
        except ValueError as e:
            refused += 1
            assert 'overlap' in str(e)
            continue
        taken += 1
        assert apart, (q.shape, k.shape, strides, places)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert taken > 50 and refused > 50, (taken, refused)


@pytest.mark.parametrize('type,shift', [(torch.float16, 3), (torch.float32, 1), (torch.bfloat16, 4), (torch.float16, 8)])
@pytest.mark.parametrize('part', [64, 20])
def test_what_lies_around_stays(device, type, shift, part):
    """The values before and behind the rows, at any alignment, in place and apart (where a product and a sum are fused may differ between
    alignments, so both are at the same one)."""
    announce('rotary around', type, shift, part)
    flat = torch.randn(shift + 2 * 5 * 12 * D + 16, generator=torch.Generator().manual_seed(5)).to(type).to(device)
    other, before = torch.full_like(flat, 3.0), flat.clone()
    slices = [t[shift:-16].view(2, 5, 12, D) for t in (flat, other)]
    (q, k), (out, out_k) = ((t[:, :, :9], t[:, :, 9:]) for t in slices)
    rotary, position = rotary_of(device, part), torch.tensor([100, 7], device=device)
    lb.rotary(q, position, rotary, k=k, out=out, out_k=out_k)
    assert torch.equal(flat, before)
    lb.rotary(q, position, rotary, k=k, out=q, out_k=k)
    assert torch.equal(slices[0], slices[1]) and not torch.equal(flat, before)
    assert torch.equal(flat[:shift], before[:shift]) and torch.equal(flat[-16:], before[-16:])
    assert bool((other[:shift] == 3).all()) and bool((other[-16:] == 3).all())
