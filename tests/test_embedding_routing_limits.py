"""The embedding and routing entry points at the largest sizes they accept and just beyond, as far as the host decides them: no GPU needed."""
import ctypes as C

import pytest

from loops_amd import _lib

F32, F16, BF16, I32, I64 = 0, 1, 2, 0, 1
BADARG, RANGE = -1, -2
MOST = 2 ** 31 - 4097  # tokens (times choices) that routing accepts


def _bytes(name, *args):
    size = C.c_size_t(0)
    code = getattr(_lib.lib(), name)(*args, C.byref(size))
    assert code == 0, (name, args, code)
    return size.value


@pytest.mark.parametrize("tokens", [2 ** 31 - 2 ** 22 - 10 ** 6, 2143293000, 2143293440, 2143303440, 2 ** 31 - 5000, MOST])
def test_workgroups_share_out_every_token(tokens):
    """512 workgroups of tokens / 512 each, rounded up, take all tokens; a workspace of 0 bytes would say that there is one workgroup."""
    per = -(-tokens // 512)
    groups = -(-tokens // per)
    experts = 16
    assert _bytes("loops_expert_counts_workspace", tokens, 1, experts) == groups * experts * 4
    assert _bytes("loops_balance_loss_workspace", tokens, experts) == (groups * (2 * 64 + 1) + 1 + 1) * 4
