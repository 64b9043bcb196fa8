"""The plain operators on drafted tokens at the edges of what they accept, on the CPU."""
import pytest
import torch

from rag_tl_domainllm_optimizer_amd import models, ops
from rag_tl_domainllm_optimizer_amd.generation import KVCache


def _i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32)


# ------------------------------------------------------------------------------------------ rows wider than they need
@pytest.mark.parametrize("extra", [1, 4, 8, 12])
@pytest.mark.parametrize("told", [False, True])
def test_accept_of_rows_with_further_columns(extra, told):
    """the rows that tree_attention read, with columns behind [q | k | v]: the same keys and values are appended as from rows without"""
    B, N, L, Hq, Hkv, D, slots = 2, 3, 2, 2, 1, 4, 9
    tokens = torch.arange(N).repeat(B, 1)
    wide = [torch.randn(B * N, (Hq + 2 * Hkv) * D + extra, generator=torch.Generator().manual_seed(i)) for i in range(L)]
    out = []
    for rows in ([x[:, :(Hq + 2 * Hkv) * D] for x in wide], wide):
        kc, vc = (torch.zeros(L, B, Hkv, slots, D) for _ in "kv")
        tree = ops.draft_tree(_i32([[-1, 0, 1]] * B))
        if not told:
            ops.tree_attention(rows[0], kc[0], vc[0], _i32([5, 0]), tree, Hq)
        out.append([*ops.tree_accept(tree, tokens, (tokens + 1) % N, rows, kc, vc, _i32([5, 0]), **(dict(Hq=Hq) if told else {})), kc, vc])
    assert out[0][0].tolist() == [N, N]
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cols,Hkv,Hq", [(17, 1, None), (28, 2, None), (16, 1, 3), (16, 1, 0), (16, 1, -2), (28, 2, 3), (8, 1, None)])
def test_accept_refuses_rows_that_do_not_hold_the_heads(cols, Hkv, Hq):
    with pytest.raises(ValueError):
        ops.tree_accept(ops.draft_tree(_i32([[-1, 0]])), *(torch.zeros(1, 2, dtype=torch.int64) for _ in "tc"), [torch.zeros(2, cols)],
                        *(torch.zeros(1, 1, Hkv, 9, 4) for _ in "kv"), _i32([3]), Hq=Hq)
