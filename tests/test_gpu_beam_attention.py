"""Decode attention over pages with their own scales: the choice between whole and cut sequences, and the bits that scores and weights keep."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("B,L,H,hkv,d,name,cut", [(40, 600, 14, 2, 64, "fp32", False), (100, 1000, 14, 2, 64, "fp32", True), (50, 900, 28, 4, 128, "fp32", True),
                                                  (60, 700, 24, 2, 128, "bf16", False), (30, 2000, 24, 2, 128, "bf16", True), (4, 519, 14, 2, 64, "bf16", True),
                                                  (58, 575, 32, 8, 128, "bf16", False)])
def test_sequences_are_cut_by_the_ctas_that_the_launch_has(cuda, B, L, H, hkv, d, name, cut):
    """A kv head's query heads may take several CTAs (8 of bf16, 4 of fp32 each), which leaves fewer ranges.  Parts of cut sequences are what the
    workspace is written for."""
    from tests.test_gpu_beams import make_kv
    from transformer_surgeon_b200 import ops
    kv = make_kv(B, (L + 15) // 16, hkv, d, cuda, lens=[L] * B)
    ws = torch.zeros(ops.decode_attn_workspace_bytes(B, H, d, L), dtype=torch.uint8, device=cuda)
    ops.paged_decode_attention(kv, torch.ones(B, H, d, dtype=DT[name], device=cuda), L, ws=ws)
    assert bool(ws[ops.COUNTER_BYTES:].any()) == cut
