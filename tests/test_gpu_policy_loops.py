"""The learned-policy operators where their loops come round: second and later rows of a warp, refilled rings, several
launches of a table, many CTAs over a long axis, and episodes that start at a chunk's edge.

Bounds and restatements are those of test_gpu_policy.py.
"""
import math

import pytest

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu

from gpu_libero_b200 import policy  # noqa: E402
from test_gpu_policy import DTYPES, check_attention, check_clip, check_norm, close, close_rows, generator, inputs  # noqa: E402


# ---- layer norm ---------------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('width', [40, 111, 257, 600, 771, 1024])
@pytest.mark.parametrize('pad', [0, 5])
def test_norm_many_rows(dtype, width, pad):
    """Every warp (group, for narrow rows) takes several rows, through more of them than its ring holds at once."""
    g = generator(width)
    rows = 20011
    wide = (torch.randn((rows, width + pad), generator=g, device='cuda') * 1.5 + 0.3).to(dtype)
    dy = torch.randn((rows, width), generator=g, device='cuda').to(dtype)
    w, b = 1 + 0.2 * torch.randn(width, generator=g, device='cuda'), 0.1 * torch.randn(width, generator=g, device='cuda')
    x = wide[:, pad:].detach()
    y, got = check_norm(x, w, b, dy)
    again = check_norm(x, w, b, dy)[1]
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [15, 16, 17])
@pytest.mark.parametrize('width', [257, 771, 1024])
def test_norm_a_handful_of_rows(dtype, rows, width):
    """One CTA takes up to 16 rows and its sums are the gradients: a warp's fourth row is past its ring."""
    g = generator(rows)
    x = torch.randn((rows, width), generator=g, device='cuda').to(dtype)
    dy = torch.randn((rows, width), generator=g, device='cuda').to(dtype)
    w = (1 + 0.2 * torch.randn(width, generator=g, device='cuda')).to(dtype)
    check_norm(x, w, torch.zeros_like(w), dy)


# ---- clipping -----------------------------------------------------------------
@pytest.mark.parametrize('count', [96, 97, 999, 1001, 2003])
@pytest.mark.parametrize('in_place', [False, True])
def test_clip_tables(count, in_place):
    """A small table, a large one, and more tensors than one launch's table holds."""
    g = generator(count)
    sizes = torch.randint(1, 3000, (count,), generator=torch.Generator().manual_seed(count)).tolist()
    grads = [torch.randn(n, generator=g, device='cuda').to(DTYPES[i % 3]) for i, n in enumerate(sizes)]
    check_clip(grads, 2.0, in_place)


# ---- decay attention ----------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('batch', [147, 150, 300])
def test_attention_many_long_rows(dtype, batch):
    """Around as many CTAs as SMs, each with a long row: the last number that is split, and the first ones that are not."""
    t = inputs(batch, 700, 1, 1, 32, 32, dtype, episode=200, ragged=True, seed=batch)
    check_attention(t, close=close_rows)


EDGES = [0, 1, 15, 16, 31, 32, 33, 62, 63, 64, 65, 126, 127, 128, 129, 191, 192, 255, 256, 257]


@pytest.mark.parametrize('dtype,time,width', [(torch.float32, 300, 40), (torch.float16, 300, 64), (torch.bfloat16, 300, 64),
                                              (torch.bfloat16, 300, 33), (torch.bfloat16, 1200, 128)])
def test_attention_episodes_at_every_edge(dtype, time, width):
    """One start a row, at and beside every edge of a chunk; rows that end at, before and behind their start."""
    batch = 3 * len(EDGES)
    t = inputs(batch, time, 1, 1, width, width, dtype, seed=width)
    t['first'] = torch.zeros((batch, time), dtype=torch.bool, device='cuda')
    at = torch.tensor(EDGES * 3, device='cuda')
    t['first'][torch.arange(batch, device='cuda'), at] = True
    t['lengths'] = torch.cat([at[:len(EDGES)], at[:len(EDGES)] + 1, at[:len(EDGES)] * 0 + time]).int()
    check_attention(t, close=close_rows)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('time,heads,kv_heads,dk,dv', [(150, 2, 2, 64, 64), (150, 4, 2, 40, 24), (150, 2, 1, 33, 31),
                                                       (150, 2, 2, 128, 96), (2000, 1, 1, 64, 64), (2000, 1, 1, 128, 128)])
@pytest.mark.parametrize('bad', [math.nan, math.inf])
def test_attention_gradients_survive_poison_before_an_episode(dtype, time, heads, kv_heads, dk, dv, bad):
    """A world that diverged and was reset: its later episode has the gradients that it has without, and so do the
    queries before it diverged."""
    start = time // 2 + 2
    t = inputs(2, time, heads, kv_heads, dk, dv, dtype, seed=dk)
    t['first'] = torch.zeros((2, time), dtype=torch.bool, device='cuda')
    t['first'][:, start] = True
    dout = torch.randn((2, time, heads, dv), generator=generator(1), device='cuda').to(dtype)

    def both(u):
        leaves = [u[n].detach().requires_grad_() for n in ('q', 'k', 'v', 'state')]
        out, state = policy.decay_attention(**dict(u, **dict(zip(('q', 'k', 'v', 'state'), leaves))))
        return (out, *torch.autograd.grad((out, state), leaves, (dout, torch.ones_like(state)))[:3]), state

    want, want_state = both(t)
    spoilt = {n: x.clone() if torch.is_tensor(x) else x for n, x in t.items()}
    for n in 'qkv':
        spoilt[n][:, start - 7:start] = bad
    got, got_state = both(spoilt)
    close(got_state, want_state.double(), time)
    for x, y in zip(got, want):
        close_rows(x[:, start:], y[:, start:].double(), 2 * time)
    for x, y in zip(got[:2], want[:2]):  # (keys and values before it feed the diverged tokens)
        close_rows(x[:, :start - 7], y[:, :start - 7].double(), 2 * time)
