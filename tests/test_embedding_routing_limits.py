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


@pytest.mark.parametrize("grad_type,out_type,width", [(BF16, F32, 4), (F16, F16, 8), (F32, F32, 4)])
@pytest.mark.parametrize("tokens", [1, 100, 5000])
def test_gradient_workspace_of_the_widest_rows(grad_type, out_type, width, tokens):
    """Rows are worked on 2^27 columns at a time: the workspace is that of as many columns, whatever the whole width, up to 2^31 - 1."""
    columns = 2 ** 27
    slabs = columns // (64 * width)
    items = max(16, -(-tokens * slabs // 16384))
    tiles = -(-tokens // items)
    bytes_of = lambda dim: _bytes("loops_embedding_gradient_workspace", grad_type, out_type, tokens, 7, dim, 0)  # noqa: E731
    want = -(-tiles * 8 // 256) * 256 + 2 * tiles * columns * 4
    assert bytes_of(columns) == want
    for dim in (columns + 1, columns + 100000, 2 ** 31 - 600, 2 ** 31 - 513, 2 ** 31 - 512, 2 ** 31 - 100, 2 ** 31 - 1):
        # (the last range, narrower, may be cut into more tiles: by a tile's rounding at most)
        assert want <= bytes_of(dim) <= 2 * want, dim
    assert _bytes("loops_embedding_gradient_workspace", grad_type, out_type, 2 ** 30, 7, 2 ** 31 - 1, 0) > 0  # (more than any memory, and no overflow)


A, B, D, G, H = (1 << 40, 2 << 40, 3 << 40, 4 << 40, 5 << 40)  # addresses far apart, never read


@pytest.mark.parametrize("off", [1, 4, 8, 12])
def test_workspaces_that_are_not_16_byte_aligned_are_refused(off):
    lib, size = _lib.lib(), 1 << 40
    assert lib.loops_group_tokens(I64, 9000, A, 100, 0, -1, B, D, G + off, size, None) == BADARG
    assert lib.loops_embedding_gradient(BF16, F32, 2000, A, B, 30, 16, D, 16, 1.0, 0, G, 16, H + off, size, None) == BADARG
    assert lib.loops_expert_counts(I64, 100000, 4, A, None, 16, B, G + off, size, None) == BADARG
    assert lib.loops_balance_loss(F32, I64, 100000, 16, 4, A, 16, B, None, 1.0, D, D + 64, D + 256, D + 512, G + off, size, None) == BADARG
