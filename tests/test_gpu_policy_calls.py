"""What a call of the learned-policy operators leaves behind, and what it must not depend on."""
import pytest

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu

from gpu_libero_b200 import policy  # noqa: E402
from test_gpu_policy import close, close_rows, inputs, recurrence  # noqa: E402


# ---- writes that autograd sees -------------------------------------------------
def test_backward_refuses_a_memory_that_acting_overwrote():
    t = inputs(2, 5, 2, 2, 8, 8, torch.float32)
    t['q'].requires_grad_()
    token = [t[n].detach()[:, 0] for n in 'qkv'] + [t['log_decay']]
    out, _ = policy.decay_attention(**t)
    policy.decay_attention_step(*token, t['state'])  # into a new tensor: nothing is overwritten
    torch.autograd.grad(out.sum(), t['q'], retain_graph=True)
    policy.decay_attention_step(*token, t['state'], state_out=t['state'])
    with pytest.raises(RuntimeError, match='inplace operation'):
        out.sum().backward()


@pytest.mark.parametrize('into', [False, True])
def test_backward_refuses_values_that_clipping_overwrote(into):
    x, w = torch.randn(9, device='cuda'), torch.ones(9, device='cuda', requires_grad=True)
    y, z = (x * w).sum(), torch.randn(9, device='cuda')
    if into:
        policy.clip_grad_norm([z], 0.1, out=[x])
    else:
        policy.clip_grad_norm([x], 0.1)
    with pytest.raises(RuntimeError, match='inplace operation'):
        y.backward()


def test_writes_to_inference_tensors():
    with torch.inference_mode():
        t = inputs(2, 1, 2, 2, 8, 8, torch.float32)
        token = [t[n][:, 0] for n in 'qkv'] + [t['log_decay']]
        want = policy.decay_attention_step(*token, t['state'])[1]
        assert torch.equal(policy.decay_attention_step(*token, t['state'], state_out=t['state'])[1], want)
        g = torch.full((4,), 2.0, device='cuda')
        assert float(policy.clip_grad_norm([g], 2.0)) == 4 and bool(((g - 1).abs() < 1e-6).all())


# ---- forward mode --------------------------------------------------------------
def test_forward_mode_is_refused_and_plain_tensors_are_not():
    from torch.autograd import forward_ad
    t = inputs(2, 5, 2, 2, 8, 8, torch.float32)
    x = torch.randn((3, 8), device='cuda')
    want = policy.decay_attention(**t)[0]
    with forward_ad.dual_level():
        for n in ('q', 'k', 'v', 'state'):
            with pytest.raises(ValueError, match='forward-mode'):
                policy.decay_attention(**dict(t, **{n: forward_ad.make_dual(t[n], torch.ones_like(t[n]))}))
        with pytest.raises(ValueError, match='forward-mode'):
            policy.layer_norm(forward_ad.make_dual(x, x))
        assert torch.equal(policy.decay_attention(**t)[0], want)
    q = t['q'].clone()
    with pytest.raises(ValueError, match='forward-mode'):
        torch.func.jvp(lambda q: policy.decay_attention(**dict(t, q=q))[0], (q,), (q,))


# ---- clipping ------------------------------------------------------------------
def test_clip_refuses_shared_memory_before_it_writes():
    g = torch.randn(5000, device='cuda')
    before = g.clone()
    for grads, out in [([g, g], None), ([g[:3000], g[2999:]], None), ([g[:2000]], [g[1:2001]]),
                       ([g[:2000], g[2000:4000]], [torch.empty(2000, device='cuda'), g[:2000]])]:
        with pytest.raises(ValueError, match='share memory'):
            policy.clip_grad_norm(grads, 0.5, out=out)
    assert torch.equal(g, before)
    # neighbours in any order, and one gradient into two places, are taken
    to = [torch.empty_like(g) for _ in range(2)]
    norm = policy.clip_grad_norm([g, g], 1.0, out=to)
    want = before.double() / (2 * before.double().square().sum()).sqrt()
    assert torch.equal(to[0], to[1]) and float((to[0] - want).abs().max()) < 1e-6 and torch.equal(g, before)
    assert abs(float(norm) - float((2 * before.double().square().sum()).sqrt())) < 1e-4
    policy.clip_grad_norm([g[2500:], g[:2500]], 1.0)
    assert float((g - before.double() / before.double().norm()).abs().max()) < 1e-6


# ---- decays ---------------------------------------------------------------------
# With tokens of zero the memory only decays: every chunk of 64 tokens, and every piece
# of a long row, rounds it once more, independently (the bound that test_gpu_policy.py
# takes for n roundings of 32 bits).
@pytest.mark.parametrize('dtype,batch,heads,width,time', [
    (torch.float32, 5, 32, 8, 1 << 17), (torch.float16, 5, 32, 8, 1 << 17), (torch.bfloat16, 5, 32, 8, 1 << 17),
    (torch.float32, 1, 1, 8, 1 << 17), (torch.bfloat16, 3, 32, 128, 1 << 16), (torch.bfloat16, 1, 1, 128, 1 << 17)])
def test_attention_slow_decays_hold_over_long_rows(dtype, batch, heads, width, time):
    """Whole rows and rows in pieces, on both kernels."""
    g = torch.Generator('cuda').manual_seed(width)
    token = torch.zeros((1, 1, 1, width), dtype=dtype, device='cuda').expand(batch, time, heads, width)
    for i in range(24 // heads + 1):
        decay = -torch.linspace(1e-6 + i * 3e-8, 2e-6 + i * 3e-8, heads, device='cuda')
        state = torch.randn((batch, heads, width, width), generator=g, device='cuda')
        _, last = policy.decay_attention(token, token, token, decay, state=state)
        want = state.double() * torch.exp(decay.double() * time)[:, None, None]
        assert bool(((last - want).abs() <= 2.0 ** -24 * (8 + 4 * (time / 64) ** 0.5) * want.abs()).all())


@pytest.mark.parametrize('time', [1, 3, 64, 200, 1100])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_attention_decays_of_every_size_keep_what_is_left(dtype, time):
    """What is left of a memory is right relative to itself, however little that is."""
    decay = -torch.logspace(-7, 1, 32, device='cuda')
    for width in (8, 128):
        token = torch.zeros((2, time, 32, width), dtype=dtype, device='cuda')
        state = torch.randn((2, 32, width, width), generator=torch.Generator('cuda').manual_seed(1), device='cuda')
        want = state.double() * torch.exp(decay.double() * time)[:, None, None]
        last = policy.decay_attention(token, token, token, decay, state=state)[1]
        steps = state.clone()
        for t in range(time):
            policy.decay_attention_step(token[:, t], token[:, t], token[:, t], decay, steps, state_out=steps)
        for got in (last, steps):
            kept = want.abs() > 1e-25  # (well above what 32 bits hold)
            # exp of a rounded product of up to 70 is off by 70 * 2^-24; every step rounds twice
            bound = 2.0 ** -24 * (80 + 4 * (2 * time) ** 0.5 + 2 * time * (got is steps))
            assert float(((got - want) / want)[kept].abs().max()) <= bound


# ---- the status word --------------------------------------------------------------
@pytest.fixture
def no_word():
    """A process whose status word has not been made yet; the one that was there comes back afterwards."""
    kept = dict(policy._status_words)
    policy._status_words.clear()
    yield
    torch.cuda.synchronize()
    policy._status_words.update(kept)


def long_wide_row():
    return inputs(1, 1100, 1, 1, 128, 128, torch.bfloat16)


@pytest.mark.parametrize('made,cleared', [(True, False), (False, True), (True, True)])
def test_check_clears_a_word_of_any_mode(no_word, made, cleared):
    """Made under inference mode or not, it is cleared under the other."""
    t = long_wide_row()
    with torch.inference_mode(made):
        want = policy.decay_attention(**t)[0].clone()
    policy._status_words[torch.device('cuda:0')].data.fill_(1)  # raised by hand, as a wait that ran out would
    with torch.inference_mode(cleared):
        with pytest.raises(RuntimeError, match='gave up'):
            policy.check()
        policy.check()
    assert torch.equal(policy.decay_attention(**t)[0], want)


def test_a_call_does_not_inherit_an_earlier_ones_expired_wait():
    """The word stays raised for check(), and later calls compute all the same."""
    t = long_wide_row()
    leaves = [t[n].requires_grad_() for n in ('q', 'k', 'v', 'state')]

    def both():
        out, state = policy.decay_attention(**t)
        return (out, state, *torch.autograd.grad((out, state), leaves, (torch.ones_like(out), torch.ones_like(state))))

    want = both()
    policy.check()
    policy._status_words[torch.device('cuda:0')].fill_(1)  # raised by hand, as a wait that ran out would
    assert all(torch.equal(a, b) for a, b in zip(both(), want))
    with pytest.raises(RuntimeError, match='gave up'):
        policy.check()
    policy.check()


def test_a_capture_without_a_status_word(no_word):
    """A process whose first call is captured: the captured kernels have nothing to report, and are right."""
    t = long_wide_row()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, state = policy.decay_attention(**t)
    assert not policy._status_words
    graph.replay()
    want, want_state = recurrence(**t)
    close_rows(out, want, 1228, 'out')
    close(state, want_state, 1101, 'state')


# ---- memories ----------------------------------------------------------------------
def test_step_takes_a_strided_memory_next_to_its_output():
    t = inputs(2, 1, 2, 2, 8, 8, torch.float32)
    token = [t[n][:, 0] for n in 'qkv'] + [t['log_decay']]
    want = policy.decay_attention_step(*token, t['state'])
    store = torch.zeros(3 * 256, device='cuda')
    to, state = store[:256].view(2, 2, 8, 8), store[256:].view(2, 2, 8, 16)[..., :8]
    state.copy_(t['state'])
    got = policy.decay_attention_step(*token, state, state_out=to)
    assert got[1] is to and torch.equal(got[0], want[0]) and torch.equal(to, want[1])
    assert torch.equal(state, t['state'])


@pytest.mark.parametrize('dtype,time,width', [(torch.float32, 70, 8), (torch.float16, 70, 64), (torch.bfloat16, 70, 64),
                                              (torch.bfloat16, 1100, 128), (torch.float32, 70, 7), (torch.float32, 1, 8)])
def test_the_library_writes_memories_of_any_alignment(dtype, time, width):
    """A caller of the C ABI may put the final memory, or its gradient, at any float."""
    t = inputs(2, time, 2, 2, width, width, dtype)
    want = policy.decay_attention(**t)
    store = torch.zeros(2 * 2 * width * width + 3, device='cuda')
    for shift in (0, 1, 2, 3):
        to = store[shift:shift + 4 * width * width].view(2, 2, width, width)
        out, _ = policy._attention_forward(*(t[n] for n in ('q', 'k', 'v', 'log_decay', 'state', 'first', 'lengths', 'scale')),
                                           state_out=to)
        # (another alignment may take another kernel)
        close_rows(out, want[0].double(), time + width)
        close_rows(to, want[1].double(), time + 1)
        assert bool((store[:shift] == 0).all()) and bool((store[shift + 4 * width * width:] == 0).all())
        store.zero_()
