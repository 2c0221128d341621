"""apply_quantization's statistics and Int8Linear's attributes, without a device (the swap itself runs on CPU tensors)."""

import io

import pytest
import torch
import torch.nn as nn

from byteprof_b200.optim.skinny_linear import SkinnyLinear
from byteprof_b200.quant import select
from byteprof_b200.quant.integrate import Int8Linear, apply_quantization


def olmo():
    model = nn.Module()
    model.model = nn.Module()
    model.model.layers = nn.ModuleList([nn.ModuleDict({
        "self_attn": nn.ModuleDict({"q_proj": nn.Linear(128, 96, bias=False)}),
        "mlp": nn.ModuleDict({"down_proj": nn.Linear(256, 128, bias=False)})})])
    model.lm_head = nn.Linear(128, 64, bias=False)
    return model.to(torch.bfloat16)


@pytest.mark.parametrize("scheme,kernel,kind,reported", [
    ("int8_w8a8", "skinny", Int8Linear, None), ("int8_w8a8", "default", Int8Linear, None),
    ("int8_wo", "skinny", SkinnyLinear, "skinny"), ("int8_wo", "default", Int8Linear, None)])
def test_the_statistics_name_the_kernel_that_the_linears_run(scheme, kernel, kind, reported):
    model = olmo()
    stats = apply_quantization(model, "blocks", scheme, kernel=kernel)
    q_proj = model.model.layers[0]["self_attn"]["q_proj"]
    assert type(q_proj) is kind and stats["n_linears"] == 2 and stats.get("kernel") == reported
    assert scheme in select.VALID_SCHEMES
    if kind is Int8Linear:
        assert q_proj.act == ("int8" if scheme == "int8_w8a8" else "bf16")


def test_no_linears_report_the_kernel_asked_for():
    assert apply_quantization(olmo(), "none", "int8_wo", kernel="skinny")["kernel"] == "skinny"


def test_a_module_saved_whole_before_there_was_a_choice_of_activations_loads():
    old = Int8Linear(nn.Linear(32, 16).to(torch.bfloat16))
    del old.__dict__["act"]
    buf = io.BytesIO()
    torch.save(old, buf)
    buf.seek(0)
    back = torch.load(buf, weights_only=False)
    assert back.act == "bf16" and "GEMV" in repr(back)
    with pytest.raises(ValueError, match="CUDA"):
        back(torch.zeros(1, 32, dtype=torch.bfloat16))
