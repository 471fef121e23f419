"""DecodePlan.run refuses tensors that its kernels cannot reach: checked before anything is launched."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def plan_on(index):
    """A plan for q [2, 4, 128] on the GPU `index` whose library call fails the test."""
    from atflash import ops
    plan = ops.DecodePlan.__new__(ops.DecodePlan)
    plan.shape, plan.q_strides, plan._mid, plan._index = (2, 4, 128), (512, 128, 1), (), index
    plan.device = torch.device("cuda", index)

    def entry(*args):
        raise AssertionError("reached the library")
    plan._entry = entry
    return plan


def tensor(device, shape=(2, 4, 128), dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device=device)


@pytest.mark.parametrize("index,q,out", [(0, "cuda:0", "cpu"), (0, "cuda:0", "meta"), (1, "cuda:0", None), (1, "cuda:0", "cuda:0"),
                                         (0, "cpu", None)])
def test_tensors_elsewhere_are_refused(index, q, out):
    with FakeTensorMode():
        with pytest.raises(ValueError, match="plan's device"):
            plan_on(index).run(tensor(q), None if out is None else tensor(out))


def test_other_shapes_and_types_are_refused():
    with FakeTensorMode():
        for q, out in ((tensor("cuda:0", (2, 4, 64)), None), (tensor("cuda:0", dtype=torch.float32), None),
                       (tensor("cuda:0"), tensor("cuda:0", (2, 4, 64))), (tensor("cuda:0"), tensor("cuda:0", dtype=torch.float32)),
                       (tensor("cuda:0"), tensor("cuda:0", (2, 128, 4)).transpose(1, 2))):
            with pytest.raises(ValueError):
                plan_on(0).run(q, out)
