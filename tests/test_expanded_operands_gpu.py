"""Expanded operands through the native form of the calls: it leaves them to the Python form, which refuses. What lies behind the one item belongs to the same tensor."""
import pytest
import torch

import brodiffusion_amd as bd

pytestmark = pytest.mark.gpu


def test_expanded_operands_are_refused():
    t = torch.zeros(2, 6, 128, dtype=torch.float16, device="cuda")
    one, rows = t[:1].expand(2, 6, 128), t[:, :1].expand(2, 6, 128)
    flat = t[0, :1].expand(6, 128)
    table = torch.zeros(6, 32, device="cuda")
    gain = torch.ones(64, dtype=t.dtype, device="cuda")
    for call in (lambda: bd.sdpa_forward(t, one, t, 2), lambda: bd.sdpa_forward(t, t, one, 2), lambda: bd.sdpa_forward(rows, t, t, 2), lambda: bd.sdpa_forward(t, t, t, 2, out=torch.empty_like(t)[:1].expand(2, 6, 128)),
                 lambda: bd.sdpa_forward(t, t, t, 2, k_prefix=one, v_prefix=t), lambda: bd.flash_attention_forward(t[0], flat, t[0], None, 2, False),
                 lambda: bd.linear_attention_relu_forward(t, one, t, 4), lambda: bd.rms_norm_rows(flat, t[0, 0], 1e-6), lambda: bd.rope_apply(flat, table, table, 64, 2),
                 lambda: bd.headnorm_rope(flat, gain, 1e-6, None, None, 64, 2), lambda: bd.headnorm_rope(t[0], gain, 1e-6, None, None, 64, 2, cache_out=t[1, :1].expand(4, 128)),
                 lambda: bd.joint_attention(t[0], flat, t[0], table, table, 64, 2)):
        with pytest.raises(RuntimeError, match="expanded"):
            call()
    # one item has no stride to speak of
    assert torch.equal(bd.sdpa_forward(t[:1].expand(1, 6, 128), t[:1], t[:1], 2), bd.sdpa_forward(t[0], t[0], t[0], 2)[None])
