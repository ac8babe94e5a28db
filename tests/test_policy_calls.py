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


# ---- sizes and pointers ----------------------------------------------------------
def test_rows_too_long_to_count_are_refused():
    many = (1 << 31) - 512
    q = torch.zeros(1, 1, 1, 8).expand(1, many, 1, 8)
    with pytest.raises(ValueError, match='too many tokens'):
        policy.decay_attention(q, q, q, torch.zeros(1))
    for width in (many, 1 << 31):
        with pytest.raises(ValueError, match='too many columns'):
            policy.layer_norm(torch.zeros(2, 1).expand(2, width))


ATTENTION = ('q k v log_decay state first lengths out state_out dout dstate_out dq dk_out dv_out dstate workspace status '
             'strides batch time heads kv_heads dk dv dtype scale').split()


def attention_args(**over):
    """A B200AttentionArgs of five tokens whose pointers are all there (and none of which may ever be launched)."""
    fields = dict.fromkeys(ATTENTION[:17], 4096)
    fields.update(strides=(80, 16, 8) * 4 + (5, 1), batch=1, time=5, heads=2, kv_heads=1, dk=8, dv=8, dtype=2, scale=1.0)
    fields.update(over)
    flat = [x for n in ATTENTION for x in (fields[n] if n == 'strides' else (fields[n],))]
    return policy.native.PolicyLibrary.ATTENTION.pack(*flat)


def norm_args(**over):
    fields = dict.fromkeys('x weight bias y stats dy dx dweight dbias workspace'.split(), 4096)
    fields.update(rows=1000, x_row=96, dy_row=96, width=96, dtype=2, weight_dtype=0, eps=1e-5)
    fields.update(over)
    return policy.native.PolicyLibrary.NORM.pack(*fields.values())


@pytest.mark.parametrize('name,args', [
    *[('attention_forward', dict([(n, 0)])) for n in ('q', 'k', 'v', 'log_decay', 'out', 'state_out')],
    *[('attention_forward', dict([(n, 0), ('time', 1)])) for n in ('q', 'out', 'state_out')],
    *[('attention_backward', dict([(n, 0)])) for n in ('q', 'k', 'v', 'log_decay', 'dout', 'dq', 'dk_out', 'dv_out',
                                                       'workspace')],
    ('attention_backward', dict(workspace=4104)), ('attention_forward', dict(time=(1 << 31) - 1)),
    ('attention_forward', dict(time=4096, heads=1, workspace=0)),
    ('attention_forward', dict(time=4096, heads=1, workspace=4104)),
    *[('norm_forward', dict([(n, 0)])) for n in ('x', 'y')], ('norm_forward', dict(stats=4100)),
    ('norm_forward', dict(width=(1 << 31) - 1)),
    *[('norm_backward', dict([(n, 0)])) for n in ('x', 'dy', 'stats', 'workspace')],
    ('norm_backward', dict(stats=4100)), ('norm_backward', dict(workspace=4104))])
def test_launches_reject_what_is_not_there_or_not_aligned(name, args):
    layout = attention_args if name.startswith('attention') else norm_args
    with pytest.raises(RuntimeError, match='CUDA error 1$'):  # before any launch
        policy._lib().launch(name, layout(**args), 0)


def test_clip_rejects_missing_memory():
    for src, dst in ((0, 4096), (4096, 0)):
        with pytest.raises(RuntimeError, match='CUDA error 1$'):
            policy._lib().launch('clip', policy.native.PolicyLibrary.CLIP.pack(src, dst, 4, 0), 1, 1.0, 0.0, 256, 256, 0)


def test_values_of_one_slice_are_not_cut_in_two():
    """Wide keys with values of up to 64: one CTA a row and head, so that 80 of them are split over a long axis."""
    shape = dict(time=500, heads=4, batch=20, dk=128)
    for dtype in (1, 2):
        assert attention_workspace(**shape, dv=64, dtype=dtype) and attention_workspace(**shape, dv=40, dtype=dtype)
        for dv in (72, 96, 128):  # three slices of 32, or two of 64: more CTAs than SMs
            assert not attention_workspace(**shape, dv=dv, dtype=dtype)


@pytest.mark.parametrize('width,row,dtype,ctas', [
    (771, 1027, 0, 2), (1024, 1024, 0, 2), (513, 513, 0, 2), (512, 512, 0, 4), (256, 256, 0, 4),
    (1024, 1024, 1, 3), (771, 771, 2, 3), (512, 512, 2, 4), (256, 256, 1, 4)])
def test_norm_gradients_take_one_wave_of_ctas(width, row, dtype, ctas):
    """A partial row for each CTA: as many as an SM's shared memory holds (228 KB, 1 KB more for each CTA)."""
    args = norm_args(rows=30011, width=width, x_row=row, dy_row=width, dtype=dtype, workspace=0)
    assert policy._lib().size('norm', args) == 148 * ctas * 2 * width * 4
