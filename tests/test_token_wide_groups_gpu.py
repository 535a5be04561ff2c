"""The one-token step of groups up to the documented 32768 channels, of many
narrow heads too: a CTA holds three numbers a head beside its channels."""

from __future__ import annotations

import pytest
import torch

from test_ssm_gpu import check_token, k, run_token, token_case  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,heads,head_dim,groups,d_state", [
    (1, 16384, 2, 1, 8), (1, 32768, 1, 1, 4), (30, 32768, 1, 1, 4), (1, 65536, 1, 2, 4), (2, 128, 256, 1, 16),
    (1, 12000, 2, 1, 256), (1, 8193, 3, 1, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_wide_groups(k, cuda, seqs, heads, head_dim, groups, d_state, dtype):  # noqa: F811
    c = token_case(seqs, heads, head_dim, groups, d_state, 3, dtype, seed=heads)
    check_token(c, dtype, run_token(k, cuda, c, dtype))
