"""The paged-cache operators' torch binding: what it refuses, and what it leaves alone."""
import pytest

from test_gpu_ops import Attention, ops, rope_case, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def test_gradients_are_refused(ops, torch):
    """Inputs that require gradients, where these are recorded; not under no_grad."""
    case = Attention(torch, "f32", [5, 6], 4, 2, 64, 16)
    slopes = torch.zeros(4, device="cuda")
    rope = rope_case(torch, "f32", 3, 4, 2, 64, 64, 16)
    names = ("q", "k", "v", "keys", "values", "table", "sequences", "positions", "cos", "sin")
    logits, scores = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    own = lambda t: t.clone().requires_grad_()  # noqa: E731

    def attend(**changed):
        given = dict(q=case.q, keys=case.keys, values=case.values, slopes=slopes)
        return ops.paged_attention(table=case.table, lengths=case.n, **{**given, **changed})

    calls = [lambda name=name, t=t: attend(**{name: own(t)})
             for name, t in (("q", case.q), ("keys", case.keys), ("values", case.values),
                             ("slopes", slopes))]
    calls += [lambda name=name: ops.rope_append(*({**rope, name: own(rope[name])}[n]
                                                  for n in names))
              for name in ("q", "k", "v", "cos", "sin")]
    calls += [lambda: ops.beam_select(own(logits), scores, 3),
              lambda: ops.beam_select(logits, own(scores), 3)]
    for call in calls:
        with pytest.raises(ValueError, match="requires gradients"):
            call()
        with torch.no_grad():
            call()
    assert not attend()[0].requires_grad


def test_the_current_device_stays(gpu, torch):
    """Operators of one device, made and called while another is current."""
    from lrrt_b200 import ops as module
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    logits = torch.randn(1, 2, 500, device="cuda:1")
    scores = torch.zeros(1, 2, device="cuda:1")
    with torch.cuda.device(0):
        with module.Ops(1) as second:
            assert torch.cuda.current_device() == 0
            first = second.beam_select(logits, scores, 2)
            assert torch.cuda.current_device() == 0
            second.reserve(1 << 26, 100000)
            assert torch.cuda.current_device() == 0
            again = second.beam_select(logits, scores, 2)
        assert torch.cuda.current_device() == 0
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert torch.zeros(1, device="cuda").device.index == 0
