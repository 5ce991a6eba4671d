"""gq_rotary_f16: both layouts, parts of the head, strided and misaligned rows, far positions, the inverse as gradient."""
import numpy as np
import pytest
import torch

from operators_testlib import HALF16, TINY16, assert_within, rotate
from popxl_addons.ops.rotary_pos_embed import RotaryPosEmbed, rotary_frequencies, rotary_pos_embed

pytestmark = pytest.mark.gpu


def _rows(tokens, heads, dim, seed):
    return np.random.default_rng(seed).normal(0, 1, (tokens, heads, dim)).astype(np.float16)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,dim,rotary_dim", [(1, 1, 64, 64), (3, 16, 256, 64), (5, 7, 80, 80), (130, 3, 128, 96),
                                                         (2, 1, 6, 4), (9, 2, 72, 18), (700, 40, 128, 128), (1, 33, 256, 256)])
def test_against_64_bits(hip, device, layout, tokens, heads, dim, rotary_dim):
    t = _rows(tokens, heads, dim, tokens + dim)
    positions = np.random.default_rng(dim).integers(0, 1 << 20, tokens).astype(np.int32)
    rotary = RotaryPosEmbed(rotary_dim, layout=layout, device=device)
    got = rotary_pos_embed(torch.from_numpy(t).to(device), torch.from_numpy(positions).to(device), rotary)
    frequencies, factor = rotary_frequencies(rotary_dim)
    want, room = rotate(t, positions, frequencies, factor, layout)
    assert_within(got.cpu().numpy(), want, room)
    assert np.array_equal(got.cpu().numpy()[..., rotary_dim:], t[..., rotary_dim:])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_extreme_positions(hip, device, layout):
    positions = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31], np.int32)
    t = _rows(5, 2, 64, 1)
    got = rotary_pos_embed(torch.from_numpy(t).to(device), torch.from_numpy(positions).to(device), RotaryPosEmbed(64, layout=layout, device=device))
    want, room = rotate(t, positions, *rotary_frequencies(64), layout)
    assert np.array_equal(got[0].cpu().numpy(), t[0])
    # (2^31 positions times a frequency of 1 leaves 2^31 2^-52 / 2 pi turns to binary64's rounding: below binary32's)
    assert_within(got.cpu().numpy(), want, room + 2e-6)


@pytest.mark.parametrize("scaling", [dict(kind="linear", factor=4), dict(kind="ntk", factor=4), dict(kind="yarn", factor=8, original_length=2048)])
def test_stretched(hip, device, scaling):
    t, positions = _rows(40, 4, 128, 3), np.arange(40, dtype=np.int32) * 401
    rotary = RotaryPosEmbed(128, layout="half", scaling=scaling, device=device)
    got = rotary_pos_embed(torch.from_numpy(t).to(device), torch.from_numpy(positions).to(device), rotary)
    want, room = rotate(t, positions, *rotary_frequencies(128, scaling=scaling), "half")
    assert_within(got.cpu().numpy(), want, room)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_slices_in_place_and_misaligned(hip, device, layout, shift):
    """q and k as they lie in a fused projection's result; `shift` elements off a 16-byte border run element by element."""
    tokens, heads, dim, rotary_dim = 6, 5, 64, 32
    wide = torch.from_numpy(_rows(tokens, 1, 8 * dim + 16, 4)[:, 0]).to(device)
    before = wide.clone()
    view = wide[:, shift:shift + heads * dim].unflatten(1, (heads, dim))
    positions = torch.arange(tokens, dtype=torch.int32, device=device) * 37
    rotary = RotaryPosEmbed(rotary_dim, layout=layout, device=device)
    apart = rotary_pos_embed(view, positions, rotary)
    assert apart.is_contiguous() and torch.equal(wide, before)
    want, room = rotate(view.cpu().numpy(), positions.cpu().numpy(), *rotary_frequencies(rotary_dim), layout)
    assert_within(apart.cpu().numpy(), want, room)
    assert rotary_pos_embed(view, positions, rotary, out=view) is view
    assert torch.equal(view, apart)
    wide[:, shift:shift + heads * dim] = before[:, shift:shift + heads * dim]
    assert torch.equal(wide, before)  # nothing beside the slice was written
    by_head = view.transpose(0, 1).contiguous().transpose(0, 1)  # head-major memory
    assert torch.equal(rotary_pos_embed(by_head, positions, rotary), apart)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_inverse_is_the_gradient(hip, device, layout):
    """The map is linear: <dy, f(t + e) - f(t - e)> = 2 <f^-1(dy), e>, to the roundings of both sides."""
    scaling = dict(kind="yarn", factor=4, original_length=512)
    tokens, heads, dim = 7, 3, 64
    t, dy, e = (_rows(tokens, heads, dim, 10 + i) for i in range(3))
    positions = torch.arange(tokens, dtype=torch.int32, device=device) * 1001
    rotary = RotaryPosEmbed(48, layout=layout, scaling=scaling, device=device)
    call = lambda a, **k: rotary_pos_embed(torch.from_numpy(a).to(device), positions, rotary, **k).cpu().numpy().astype(np.float64)  # noqa: E731
    grad = call(dy, inverse=True)
    up, down = t + e, t - e  # (rounded to binary16: the step is what they differ by)
    f_up, f_down = call(up), call(down)
    left = dy * (f_up - f_down)
    right = grad * (up.astype(np.float64) - down.astype(np.float64))
    room = (np.abs(dy) * (HALF16 * 1.01 * (np.abs(f_up) + np.abs(f_down)) + 2 * TINY16)).sum()
    room += (np.abs(up.astype(np.float64) - down) * (HALF16 * 1.01 * np.abs(grad) + TINY16)).sum() + 1e-4
    assert abs(left.sum() - right.sum()) <= room
    want, allowed = rotate(dy, positions.cpu().numpy(), *rotary_frequencies(48, scaling=scaling), layout, sign=-1)
    assert_within(grad, want, allowed)


def test_values_that_are_not_finite_stay_in_their_pair(hip, device):
    t = _rows(2, 2, 64, 5)
    t[0, 0, 0], t[1, 1, 63] = np.inf, np.nan
    positions = torch.tensor([3, 4], dtype=torch.int32, device=device)
    got = rotary_pos_embed(torch.from_numpy(t).to(device), positions, RotaryPosEmbed(32, device=device)).cpu().numpy()
    bad = ~np.isfinite(got)
    assert bad[0, 0, :2].all() and np.isnan(got[1, 1, 63]) and bad.sum() == 3


def test_empty_and_other_stream(hip, device):
    rotary = RotaryPosEmbed(32, device=device)
    none = rotary_pos_embed(torch.empty((0, 4, 64), dtype=torch.float16, device=device), torch.empty(0, dtype=torch.int32, device=device), rotary)
    assert none.shape == (0, 4, 64)
    t = torch.from_numpy(_rows(33, 4, 64, 6)).to(device)
    positions = torch.arange(33, dtype=torch.int32, device=device)
    want = rotary_pos_embed(t, positions, rotary)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(device=device)
    with torch.cuda.stream(stream):
        got = rotary_pos_embed(t, positions, rotary)
    stream.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dim,tokens", [(16, 1 << 24), (2, (1 << 24) - 3)])
def test_most_tokens(hip, device, dim, tokens):
    """As many tokens as a call takes are more than a grid holds: the bits of calls on parts of them."""
    gen = torch.Generator(device=device).manual_seed(dim)
    t = torch.randn((tokens, 1, dim), generator=gen, device=device, dtype=torch.float16)
    positions = torch.randint(-2 ** 31, 2 ** 31 - 1, (tokens,), generator=gen, device=device, dtype=torch.int32)
    rotary = RotaryPosEmbed(dim, device=device)
    got, third = rotary_pos_embed(t, positions, rotary), tokens // 3
    for i in range(0, tokens, third):
        assert torch.equal(got[i:i + third], rotary_pos_embed(t[i:i + third], positions[i:i + third], rotary)), i
    assert rotary_pos_embed(t, positions, rotary, out=t) is t
    assert torch.equal(got, t)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_given_frequencies(hip, device, layout):
    t, positions = _rows(9, 3, 80, 4), np.array([0, 1, -7, 100, 2047, 65536, 3, 2 ** 31 - 1, -2 ** 31])
    w = np.random.default_rng(1).normal(0, 1, 32)
    got = rotary_pos_embed(torch.from_numpy(t).to(device), torch.tensor(positions, dtype=torch.int32, device=device),
                           RotaryPosEmbed.from_frequencies(w, 1.25, layout=layout, device=device)).cpu().numpy()
    turns = positions[:, None] * (w / (2 * np.pi))  # (reduced to a turn as the definition does, so that far positions mean the same)
    want, room = zip(*(rotate(t[i:i + 1], [1], 2 * np.pi * (turns[i] - np.rint(turns[i])), 1.25, layout) for i in range(len(t))))
    assert_within(got, np.concatenate(want), np.concatenate(room))
