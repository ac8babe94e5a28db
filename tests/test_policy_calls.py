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
