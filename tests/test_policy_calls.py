"""CPU tests of what the learned-policy operators' calls refuse, and of what they must not refuse.

A call that nothing but the device keeps from running ends with the message that asks for CUDA tensors.
"""
import pytest

torch = pytest.importorskip('torch')

from torch.autograd import forward_ad  # noqa: E402

from gpu_libero_b200 import policy  # noqa: E402


def test_forward_mode_derivatives_are_refused():
    q, k, v = torch.ones(2, 3, 4, 8), torch.ones(2, 3, 2, 8), torch.ones(2, 3, 2, 6)
    decay, state, x, w = torch.zeros(4), torch.ones(2, 4, 8, 6), torch.ones(4, 6), torch.ones(6)
    calls = [(lambda q, k, v, d, s: policy.decay_attention(q, k, v, d, state=s), (q, k, v, decay, state)),
             (lambda q, k, v, d, s, to: policy.decay_attention_step(q, k, v, d, s, state_out=to),
              (q[:, 0], k[:, 0], v[:, 0], decay, state, torch.ones_like(state))),
             (policy.layer_norm, (x, w, w.clone())),
             (lambda a, b: policy.clip_grad_norm([a, None, b], 1.0), (x, w)),
             (lambda a, b: policy.clip_grad_norm([a], 1.0, out=[b]), (x, x.clone()))]
    with forward_ad.dual_level():
        for call, args in calls:
            for i in range(len(args)):
                dual = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(ValueError, match='forward-mode'):
                    call(*args[:i], dual, *args[i + 1:])
            with pytest.raises(ValueError, match='CUDA'):
                call(*args)
    for call, args in calls:
        with pytest.raises(ValueError, match='CUDA'):
            call(*args)


# ---- memory that clipping writes through one tensor and touches through another -----
def clipping_that_shares_memory():
    g, h = torch.ones(64), torch.ones(8, 8)
    return [('a gradient twice in place', [g, h, g], None),
            ('overlapping views in place', [g[:40], g[39:]], None),
            ('one inside the other', [g, g[8:16]], None),
            ('two gradients into one', [g, h.view(64)], [torch.ones(64)] * 2),
            ('into its own, shifted', [g[:32]], [g[1:33]]),
            ("into another's gradient", [g[:32], g[32:]], [torch.ones(32), g[:32]]),
            ('many tensors', [torch.ones(3) for _ in range(150)] + [g, g[63:]], None)]


@pytest.mark.parametrize('name,grads,out', clipping_that_shares_memory())
def test_clip_refuses_shared_memory(name, grads, out):
    with pytest.raises(ValueError, match='share memory'):
        policy.clip_grad_norm(grads, 1.0, out=out)
    table = b''.join(policy.native.PolicyLibrary.CLIP.pack(a.data_ptr(), b.data_ptr(), a.numel(), 0)
                     for a, b in zip(grads, out or grads))
    with pytest.raises(RuntimeError, match='CUDA error 1$'):  # before any launch
        policy._lib().launch('clip', table, len(grads), 1.0, 0.0, 256, 256, 0)


def test_clip_takes_neighbours_and_shared_sources():
    g = torch.ones(64)
    for grads, out in [([g[:32], g[32:]], None), ([g[32:], g[:32]], [g[32:], g[:32]]), ([g, g], [torch.ones(64), torch.ones(64)]),
                       ([g, g[3:9]], [torch.ones(64), torch.ones(6)]), ([g[:0], g, g[5:5]], None), ([g[:32]], [g[32:]])]:
        with pytest.raises(ValueError, match='CUDA'):
            policy.clip_grad_norm(grads, 1.0, out=out)


# ---- what the library plans ---------------------------------------------------------
def attention_workspace(time, heads, dk, dv, dtype=2, batch=1, kv_heads=None, backward=0, status=0):
    """Bytes that the library asks for a forward or backward pass over dense, aligned tensors."""
    kv_heads = kv_heads or heads
    rows = lambda heads, width: (time * heads * width, heads * width, width)  # noqa: E731
    args = policy.native.PolicyLibrary.ATTENTION.pack(
        *[256] * 4, 0, 0, 0, *[256] * 8, 0, status, *rows(heads, dk), *rows(kv_heads, dk), *rows(kv_heads, dv),
        *rows(heads, dv), 0, 0, batch, time, heads, kv_heads, dk, dv, dtype, 1.0)
    return policy._lib().size('attention', args, backward)


def test_bounded_waits_need_a_status_word():
    """The kernel with bounded waits splits a long row into pieces of one CTA an SM, the other one of several:
    without a word to report to, the other one runs."""
    with_word, without = (attention_workspace(8192, 8, 128, 128, status=s) for s in (256, 0))
    assert with_word and without > 1.5 * with_word
    # where no kernel has such waits, the word changes nothing
    for over in (dict(dtype=1), dict(dk=64, dv=64), dict(time=1000)):
        shape = dict(dict(time=8192, heads=8, dk=128, dv=128), **over)
        assert attention_workspace(**shape, status=256) == attention_workspace(**shape)


def test_clip_takes_layouts_that_differ_by_single_elements_only():
    """A 1 x 1 convolution's gradient: the dense order and the channels-last one are the same memory."""
    g = torch.ones(4, 6, 1, 1)
    alike = torch.empty(4, 6, 1, 1).to(memory_format=torch.channels_last).as_strided((4, 6, 1, 1), (6, 1, 6, 6))
    assert g.stride() != alike.stride()
    for grads, out in (([g], [alike]), ([alike], [g]), ([torch.ones(1, 5)], [torch.ones(5, 1).t()]),
                       ([torch.ones(2, 0, 5)], [torch.ones(0, 2, 5).transpose(0, 1)])):
        with pytest.raises(ValueError, match='CUDA'):
            policy.clip_grad_norm(grads, 1.0, out=out)
    with pytest.raises(ValueError, match='out must match'):
        policy.clip_grad_norm([torch.ones(4, 6)], 1.0, out=[torch.ones(6, 4).t()])
