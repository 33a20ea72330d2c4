"""What a captured training step takes: its own batch's shapes, and its teacher's types."""

from __future__ import annotations

import pytest
import torch

from omniwave_b200 import distill_loss
from omniwave_b200.train import TrainStep


class _Graph:
    """Stands for a captured graph."""

    replays = 0

    def replay(self):
        self.replays += 1


def _captured(teacher):
    step = TrainStep(torch.nn.Linear(6, 5), cuda_graph=False)
    held = [torch.zeros(4, 6), torch.zeros(4, dtype=torch.int64)]
    if teacher:
        held += [torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)]
    step._graph, step._graph_warmup, step._static = _Graph(), 0, (tuple(held), torch.zeros(()))
    return step


X, Y, TOP, CLS = torch.ones(4, 6), torch.ones(4, dtype=torch.int64), torch.ones(4, 3), torch.ones(4, 3, dtype=torch.int32)


@pytest.mark.parametrize("x,y,top,cls,match", [
    (X, Y, TOP[:, :1], CLS[:, :1], "top_logits"),      # one entry would be spread over all
    (X, Y, TOP[:, :1], CLS, "top_logits"),
    (X, Y, TOP, CLS[:, :1], "top_classes"),
    (X, Y, TOP[:1], CLS[:1], "top_logits"),
    (X, Y, TOP, CLS[0], "top_classes"),
    (X[:1], Y, TOP, CLS, "images"),
    (X, Y[:1], TOP, CLS, "labels"),
    (X, Y, TOP.bfloat16(), CLS, "top_logits in"),
    (X, Y, TOP, CLS.long(), "top_classes in"),         # a class past 2^32 would become another
])
def test_a_captured_step_refuses_other_shapes_and_types_of_a_teacher(x, y, top, cls, match):
    step = _captured(True)
    with pytest.raises(ValueError, match=match):
        step.step(x, y, teacher=(top, cls))
    assert step._graph.replays == 0 and step._nsteps == 0 and all((t == 0).all() for t in step._static[0])
    step.step(X, Y, teacher=(TOP, CLS))
    assert step._graph.replays == 1 and all((t == 1).all() for t in step._static[0])


def test_a_captured_step_refuses_other_shapes_without_a_teacher():
    step = _captured(False)
    for x, y in ((X[:1], Y), (X, Y[:1]), (X[:1], Y[:1]), (X[:, :1], Y)):
        with pytest.raises(ValueError, match="captured with"):
            step.step(x, y)
    step.step(X.double(), Y.int())  # a batch is still cast, as it was
    assert step._graph.replays == 1 and all((t == 1).all() for t in step._static[0])


@pytest.mark.gpu
def test_a_captured_step_with_teachers_of_other_lengths(cuda_device):
    torch.manual_seed(3)
    x, y = torch.randn(8, 20, device=cuda_device), torch.randint(50, (8,), device=cuda_device)
    top, cls = (torch.randn(8, 50, device=cuda_device) * 2).topk(32, 1)
    net = torch.nn.Linear(20, 50).to(cuda_device)
    kept = [p.detach().clone() for p in net.parameters()]
    step = TrainStep(net, optimizer="fused", cuda_graph=True, graph_warmup=1, amp_dtype=None, distill_weight=1.0, distill_temperature=2.0)
    for _ in range(2):
        step.step(x, y, teacher=(top, cls))
    for k in (1, 16):
        with pytest.raises(ValueError, match="captured with top_logits"):
            step.step(x, y, teacher=(top[:, :k], cls[:, :k]))
    # padded to the length that was captured, a shorter teacher gives its own loss
    with torch.no_grad():
        for p, q in zip(net.parameters(), kept):
            p.copy_(q)
        want = distill_loss(net(x), top[:, :1].contiguous(), cls[:, :1].contiguous(), y, temperature=2.0, weight=1.0)
    one = cls.clone()
    one[:, 1:] = -1
    got = step.step(x, y, teacher=(top, one))
    assert abs(got.item() - want.item()) <= 1e-5 * abs(want.item())  # about 16 u a term, of products in another order
