"""CPU: the adapters' calls and the gradients of the MoE steps refuse tensors of two devices, whose kernels would read addresses of another
GPU. The tensors are stand-ins without memory; a refused call reads none."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


def _tensors(**shapes):
    with FakeTensorMode():
        return {name: torch.empty(*shape, dtype=dtype, device="cuda:0") for name, (shape, dtype) in shapes.items()}


def _moved(t):
    with FakeTensorMode():
        return torch.empty(tuple(t.shape), dtype=t.dtype, device="cuda:1")


F, I = torch.float32, torch.int32
APPLY = dict(out=((4, 32), BF), base=((4, 32), BF), x=((4, 64), BF), a=((2, 8, 64), BF), b=((2, 32, 8), BF), scales=((2,), F),
             sorted_ids=((4,), I), offsets=((4,), I), h=((4, 8), F))
BACKWARD = dict(d_x=((4, 64), BF), d_a=((2, 8, 64), BF), d_b=((2, 32, 8), BF), d_x_base=((4, 64), BF), d_out=((4, 32), BF), x=((4, 64), BF),
                h=((4, 8), F), a=((2, 8, 64), BF), b=((2, 32, 8), BF), scales=((2,), F), sorted_ids=((4,), I), offsets=((4,), I),
                workspace=((4096,), torch.uint8))
CALLS = [("lora", "plan", dict(adapter_ids=((4,), I), sorted_ids=((4,), I), offsets=((4,), I)), dict(num_adapters=2), "adapter_ids"),
         ("lora", "apply", APPLY, {}, "x"),
         ("lora", "backward", BACKWARD, {}, "x"),
         ("moe", "unpermute_backward", dict(d_permuted=((8, 8), BF), d_weights=((4, 2), F), d_out=((4, 8), BF), permuted=((8, 8), BF),
                                            sorted_token_ids=((8,), I), routing_weights=((4, 2), F)), dict(num_tokens=4, top_k=2, hidden=8), "permuted"),
         ("moe", "permute_backward", dict(d_input=((4, 8), BF), d_permuted=((8, 8), BF), sorted_token_ids=((8,), I)),
          dict(num_tokens=4, top_k=2, hidden=8), "d_permuted"),
         ("moe", "gate_softmax_topk_backward", dict(d_logits=((4, 8), F), d_weights=((4, 2), F), weights=((4, 2), F), indices=((4, 2), I),
                                                    logits=((4, 8), F)), dict(num_tokens=4, num_experts=8, top_k=2), "d_logits")]


@pytest.mark.parametrize("module,name,shapes,sizes,reference", CALLS, ids=[c[1] for c in CALLS])
def test_tensors_of_another_device(ks, module, name, shapes, sizes, reference):
    call = getattr(getattr(ks, module), name)
    tensors = _tensors(**shapes)
    for other in shapes:
        if other == reference:
            continue
        with pytest.raises(ValueError, match=f"{other} must be on cuda:0"):
            call(**{**tensors, other: _moved(tensors[other])}, **sizes)
