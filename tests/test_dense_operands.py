"""The operators on dense q, k and v refuse parts of a fused projection, whose
rows they would read as if dense (CPU: the check runs before any GPU call)."""
import pytest
import torch

from glt_amd import ops


def parts(B=2, T=5, Hq=4, Hkv=2):
    qkv = torch.zeros((B, T, Hq + 2 * Hkv, 128), dtype=torch.bfloat16)
    return qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]


def test_rope_refuses_views():
    q, k, _ = parts()
    for a, b in ((q, k), (q, None), (q.contiguous(), k), (q, k.contiguous())):
        with pytest.raises(ValueError, match="contiguous"):
            ops.apply_rope(a, b, 10000.0)


def test_attention_refuses_views():
    x = parts()
    for i in range(3):
        with pytest.raises(ValueError, match="contiguous"):
            ops.attention(*(t if j == i else t.contiguous() for j, t in enumerate(x)))
