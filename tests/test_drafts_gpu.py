"""The kernels on drafted tokens against their 64-bit forms: sizes, masks and lengths where they can go wrong, and how they are called."""
import math
import random

import pytest
import torch

import drafts_common as plain
from rag_tl_domainllm_optimizer_amd import models, ops
from rag_tl_domainllm_optimizer_amd.generation import KVCache
from rag_tl_domainllm_optimizer_amd.runtime import GraphRunner

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def _i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


def _rand(*shape, dtype=BF16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


# ------------------------------------------------------------------------------------------ the plan
@pytest.mark.parametrize("rows,nodes", [(1, 1), (3, 2), (5, 17), (64, 64), (300, 33)])
def test_plan(rows, nodes):
    parents = plain.trees(rows, nodes, rows)
    parents[0] = [-1] + list(range(nodes - 1))
    counts = [(7 * i) % (nodes + 1) for i in range(rows)]
    counts[0] = nodes
    pos0 = list(range(rows))
    a, b = ops.draft_tree(_i32(parents), _i32(counts), _i32(pos0)), ops.draft_tree(*(torch.tensor(x, dtype=torch.int32) for x in (parents, counts, pos0)))
    assert torch.equal(a.see.cpu(), b.see) and torch.equal(a.pos.cpu(), b.pos)


def test_plan_of_odd_parents():
    parents = [[4, 1, 0, -7, 3, 99, 2 ** 31 - 1, -2 ** 31]]
    a, b = ops.draft_tree(_i32(parents)), ops.draft_tree(torch.tensor(parents, dtype=torch.int32))
    assert torch.equal(a.see.cpu(), b.see) and torch.equal(a.pos.cpu(), b.pos)


# ------------------------------------------------------------------------------------------ attention
def _attention(Hq, Hkv, D, N, lens, slots, starts=None, counts=None, window=0, dtype=BF16, seed=0, extra=0, junk=math.nan, fp8=False):
    B = len(lens)
    counts = counts or [N] * B
    parents = plain.trees(B, N, seed)
    qkv = _rand(B * N, (Hq + 2 * Hkv) * D + extra, dtype=dtype, seed=seed)
    kc, vc = (_rand(B, Hkv, slots, D, dtype=dtype, seed=seed + k) for k in (1, 2))
    for b in range(B):  # what no node sees
        for c in (kc, vc):
            c[b, :, lens[b]:] = junk
            if starts:
                c[b, :, :starts[b]] = junk
        qkv[b * N + counts[b]:(b + 1) * N] = junk
    out = torch.full((B * N, Hq * D), 7.0, dtype=dtype, device=DEV)
    tree = ops.draft_tree(_i32(parents), _i32(counts))
    held, scales = (kc, vc), {}
    if fp8:
        (kq, ks), (vq, vs) = (ops.kv_quantize_rows(c.nan_to_num(), k) for c, k in ((kc, True), (vc, False)))
        kc, vc = ops.kv_dequantize(kq, ks, True), ops.kv_dequantize(vq, vs, False)
        for b in range(B):
            for c, sc in ((kq, ks), (vq, vs)):  # no numbers where nothing is seen
                c[b, :, lens[b]:], sc[b, :, lens[b]:] = 0x7f, math.nan
                if starts:
                    c[b, :, :starts[b]], sc[b, :, :starts[b]] = 0x7f, math.nan
        held, scales = (kq, vq), dict(k_scale=torch.nn.functional.pad(ks, (0, 5)), v_scale=torch.nn.functional.pad(vs, (0, 5)))
    ops.tree_attention(qkv, *held, _i32(lens), tree, Hq, _i32(starts), window, out=out, **scales)
    want, size = plain.attention(torch.nan_to_num(qkv), kc, vc, lens, parents, counts, Hq, starts, window)
    # the output's rounding, half a step of its value; p rounded to the cache's type in front of the product with v, half a step
    # of each term; fp32 scores: D products and sums of 2^-24 each of sum |q k| scale (below 16 here), which p takes over as a
    # relative error; as much again for the sums over the keys, exp2 and the division
    half = torch.finfo(dtype).eps / 2
    fp32 = 2 * 2 ** -24 * (16 * D + sum(lens) / len(lens) + N + 64)
    tol = half * want.abs() + ((half if dtype == BF16 else 0) + fp32) * size * (1 + half)
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol.clamp(min=1e-30)).max().item():.2f} of the tolerance"


HEADS = [(4, 2, 64), (32, 8, 128), (12, 12, 64), (5, 5, 128), (16, 2, 64), (8, 1, 128), (3, 1, 32), (2, 2, 80)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("N", [1, 3, 16, 17, 64])
def test_attention(Hq, Hkv, D, N):
    _attention(Hq, Hkv, D, N, [130, 0, 1, 64], 200, seed=N)


@pytest.mark.parametrize("lens", [[0], [1], [31], [32], [33], [63, 65], [127, 128, 129], [255, 257], [500, 3, 0, 77]])
def test_attention_context_lengths(lens):
    _attention(8, 2, 128, 6, lens, max(lens) + 1)


@pytest.mark.parametrize("Hq,Hkv,D,N", [(8, 2, 128, 5), (4, 4, 64, 40), (3, 1, 32, 4)])
def test_attention_pads_and_fewer_nodes(Hq, Hkv, D, N):
    _attention(Hq, Hkv, D, N, [150, 70, 64, 33, 9], 160, starts=[3, 69, 64, 0, 8], counts=[N, 0, 1, N - 1, N])


@pytest.mark.parametrize("window", [1, 2, 5, 64, 100, 1000])
@pytest.mark.parametrize("Hq,Hkv,D,N", [(8, 2, 128, 20), (4, 4, 64, 3), (3, 1, 32, 9)])
def test_attention_window(Hq, Hkv, D, N, window):
    _attention(Hq, Hkv, D, N, [300, 20, 0, 101], 310, starts=[0, 4, 0, 50], window=window, junk=3.0)


@pytest.mark.parametrize("window", [0, 3, 40])
@pytest.mark.parametrize("N", [1, 31, 32, 63, 64])
def test_attention_last_keys_beside_the_nodes(N, window):
    """what is left of the context behind whole stages of 64 keys, beside the nodes, at and around the place where both fill a stage"""
    lens = [n for rest in (0, 1, 63 - N, 64 - N, 65 - N, 63) for n in (rest, 64 + rest) if n >= 0]
    _attention(4, 2, 64, N, lens, 200, window=window, junk=math.nan if not window else 5.0, starts=[n // 7 for n in lens] if N % 2 else None, seed=N)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_keeps_windows_apart(bad):
    """a value that is no number at the end of the context reaches the nodes whose window holds it, and no other"""
    N, window, n = 9, 4, 40  # node i at position n + i of a chain sees the slots from n + i - 3
    qkv, kc, vc = _rand(N, 8 * 64), _rand(1, 2, 50, 64, seed=1), _rand(1, 2, 50, 64, seed=2)
    tree = ops.draft_tree(_i32([[-1] + list(range(N - 1))]))
    want = ops.tree_attention(qkv, kc, vc, _i32([n]), tree, 4, window=window)
    vc[0, :, n - 2, 5] = bad
    got = ops.tree_attention(qkv, kc, vc, _i32([n]), tree, 4, window=window)
    assert torch.equal(got[2:], want[2:])
    of = got[:2].view(2, 4, 64)
    assert not torch.isfinite(of[:, :, 5]).any() and torch.isfinite(of[:, :, :5]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Hq,Hkv,D,fp8", [(2, 2, 128, False), (2, 2, 128, True), (8, 2, 128, False), (8, 2, 128, True), (8, 1, 128, False),
                                          (8, 1, 128, True), (32, 1, 128, False), (32, 1, 128, True), (4, 4, 64, False), (32, 2, 64, False),
                                          (3, 1, 32, False)])
def test_attention_windows_part_way_down_the_context(Hq, Hkv, D, fp8, bad):
    """the same far from its end, where a window of 100 starts: a value, or in e4m3 its scale, and what key and value hold before it"""
    N, window, n = 9, 100, 300  # node i at position n + i sees the slots from n + i - 99
    at = n - 95                 # seen by nodes 0 to 4
    qkv, kc, vc = _rand(N, (Hq + 2 * Hkv) * D), _rand(1, Hkv, 310, D, seed=1), _rand(1, Hkv, 310, D, seed=2)
    tree, scales = ops.draft_tree(_i32([[-1] + list(range(N - 1))])), {}
    if fp8:
        (kc, ks), (vc, vs) = ops.kv_quantize_rows(kc, True), ops.kv_quantize_rows(vc, False)
        scales = dict(k_scale=torch.nn.functional.pad(ks, (0, 2)), v_scale=torch.nn.functional.pad(vs, (0, 2)))
    run = lambda: ops.tree_attention(qkv, kc, vc, _i32([n]), tree, Hq, window=window, **scales)
    want = run()
    if fp8 and not math.isnan(bad):
        scales["v_scale"][0, :, at] = bad
        ill = slice(0, D)
    else:
        vc[0, :, at, 5] = 0x7f if fp8 else bad
        ill = slice(5, 6)
    got = run()
    assert torch.equal(got[5:], want[5:])
    of, ref = got[:5].view(5, Hq, D), want[:5].view(5, Hq, D)
    assert not torch.isfinite(of[:, :, ill]).any() and (math.isnan(bad) or fp8 or (of[:, :, ill] == bad).all())
    of[:, :, ill] = ref[:, :, ill]
    assert torch.equal(of, ref)
    (scales["k_scale"] if fp8 else kc)[0, :, at] = bad  # scores that are no numbers
    assert torch.equal(run()[5:], want[5:])


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(8, 2, 128, 64, 70), (2, 2, 128, 5, 127), (4, 4, 64, 30, 63), (3, 1, 32, 9, 20)])
def test_attention_infinite_value_at_the_end_of_the_context(Hq, Hkv, D, N, n):
    """the last slot's value stands in for keys behind it: infinite it is infinite in every node's sum, and no NaN"""
    qkv, kc, vc = _rand(N, (Hq + 2 * Hkv) * D), _rand(1, Hkv, n + 3, D, seed=1), _rand(1, Hkv, n + 3, D, seed=2)
    tree = ops.draft_tree(_i32([[-1] + list(range(N - 1))]))
    want = ops.tree_attention(qkv, kc, vc, _i32([n]), tree, Hq).view(N, Hq, D)
    vc[0, :, n - 1, 7] = math.inf
    got = ops.tree_attention(qkv, kc, vc, _i32([n]), tree, Hq).view(N, Hq, D)
    assert (got[:, :, 7] == math.inf).all()
    got[:, :, 7] = want[:, :, 7]
    assert torch.equal(got, want)


@pytest.mark.parametrize("lens", [[2100], [1500, 9, 700]])
@pytest.mark.parametrize("N", [2, 30])
def test_attention_long(lens, N):
    _attention(8, 2, 128, N, lens, max(lens) + 5)


@pytest.mark.parametrize("Hq,Hkv,D,N", [(8, 2, 128, 7), (4, 4, 64, 33), (3, 1, 20, 4)])
def test_attention_f32(Hq, Hkv, D, N):
    _attention(Hq, Hkv, D, N, [100, 0, 31], 120, dtype=F32, window=50, junk=2.0)


@pytest.mark.parametrize("Hq,Hkv,N", [(4, 4, 1), (5, 5, 16), (8, 2, 8), (32, 8, 16), (8, 2, 33), (8, 2, 64), (12, 1, 64)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_over_an_fp8_cache(Hq, Hkv, N, window):
    _attention(Hq, Hkv, 128, N, [130, 0, 1, 64, 65, 191], 200, starts=[0, 0, 0, 10, 64, 3], counts=[N, N, N, 1, N, 0], window=window, seed=N, fp8=True)


@pytest.mark.parametrize("lens", [[2100], [900, 9, 700]])
@pytest.mark.parametrize("N", [2, 30, 60])
def test_attention_over_a_long_fp8_cache(lens, N):
    _attention(8, 2, 128, N, lens, max(lens) + 5, fp8=True, extra=3 if N == 2 else 0)


@pytest.mark.parametrize("extra", [0, 3])
@pytest.mark.parametrize("N", [1, 7, 64])
def test_accept_into_an_fp8_cache(N, extra):
    r = random.Random(N)
    B, L, Hq, Hkv, D, slots = 5, 3, 4, 2, 128, 80
    parents, counts = plain.trees(B, N, N, 3), [N] + [r.randint(0, N) for _ in range(B - 1)]
    parents[0] = [-1] + list(range(N - 1))
    tokens, choice = ([[r.randrange(3) for _ in range(N)] for _ in range(B)] for _ in "tc")
    choice[0] = tokens[0][1:] + [9]
    lens = [20] + [r.randint(0, slots) for _ in range(B - 1)]
    rows = [_rand(B * N, (Hq + 2 * Hkv) * D + extra, seed=i) for i in range(L)]
    rows[0][0, Hq * D:(Hq + 1) * D] = 0  # a key of zeros
    drafts = [x[:, :(Hq + 2 * Hkv) * D] for x in rows]
    t = lambda x: torch.tensor(x)
    out = []
    for dev in ("cpu", DEV):
        kc, vc = (torch.full((L, B + 1, Hkv, slots, D), 3, dtype=torch.uint8, device=dev) for _ in "kv")
        ks, vs = (torch.full((L, B + 1, Hkv, 96), 2.0, device=dev) for _ in "kv")
        tree = ops.draft_tree(t(parents).int().to(dev), t(counts).int().to(dev))
        o = ops.tree_accept(tree, t(tokens).to(dev), t(choice).to(dev), drafts if dev == DEV else [x.cpu() for x in drafts], kc[:, :B], vc[:, :B], t(lens).int().to(dev), ks[:, :B], vs[:, :B])
        out.append([x.cpu() for x in (*o, kc, vc, ks, vs)])
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_attention_of_rows_with_an_odd_pitch():
    _attention(8, 2, 128, 9, [90, 40], 100, extra=3)
    _attention(8, 2, 128, 9, [90, 40], 100, extra=8)


def test_attention_into_columns_of_a_wider_output():
    B, N, Hq, Hkv, D = 2, 5, 4, 2, 64
    qkv, kc, vc = _rand(B * N, (Hq + 2 * Hkv) * D), _rand(B, Hkv, 50, D, seed=1), _rand(B, Hkv, 50, D, seed=2)
    tree, lens = ops.draft_tree(_i32(plain.trees(B, N, 0))), _i32([50, 20])
    want = ops.tree_attention(qkv, kc, vc, lens, tree, Hq)
    for at in (0, 8, 1):
        wide = torch.full((B * N, Hq * D + 9), 5.0, dtype=BF16, device=DEV)
        ops.tree_attention(qkv, kc, vc, lens, tree, Hq, out=wide[:, at:at + Hq * D])
        assert torch.equal(wide[:, at:at + Hq * D], want)
        assert (wide[:, :at] == 5).all() and (wide[:, at + Hq * D:] == 5).all()


def test_attention_into_other_columns_of_the_same_rows():
    B, N, Hq, Hkv, D = 2, 5, 4, 2, 64
    wide = _rand(B * N, (Hq + 2 * Hkv) * D + Hq * D)
    qkv, kc, vc = wide[:, :(Hq + 2 * Hkv) * D], _rand(B, Hkv, 50, D, seed=1), _rand(B, Hkv, 50, D, seed=2)
    tree, lens = ops.draft_tree(_i32(plain.trees(B, N, 0))), _i32([50, 20])
    want = ops.tree_attention(qkv.clone(), kc, vc, lens, tree, Hq)
    assert torch.equal(ops.tree_attention(qkv, kc, vc, lens, tree, Hq, out=wide[:, (Hq + 2 * Hkv) * D:]), want)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (3, 1, 32)])
def test_attention_keeps_nodes_apart(Hq, Hkv, D, bad):
    """keys and values that are not numbers in one branch leave the other branches as they are"""
    N = 20
    parents = [[-1, 0, 0] + list(range(1, N - 2))]  # two chains from the root: odd and even nodes
    qkv, kc, vc = _rand(N, (Hq + 2 * Hkv) * D), _rand(1, Hkv, 70, D, seed=1), _rand(1, Hkv, 70, D, seed=2)
    tree, lens = ops.draft_tree(_i32(parents)), _i32([66])
    want = ops.tree_attention(qkv, kc, vc, lens, tree, Hq)
    qkv[7, Hq * D:] = bad
    got = ops.tree_attention(qkv, kc, vc, lens, tree, Hq)
    ill = [i for i, f in enumerate(plain.chains(parents[0], N)) if 7 in f]
    well = [i for i in range(N) if i not in ill]
    assert torch.equal(got[well], want[well])
    assert torch.isnan(got[ill]).all()


def test_attention_lengths_past_the_cache_and_below_zero():
    """lengths that do not fit are cut to the cache"""
    qkv, kc, vc = _rand(6, 8 * 64), _rand(2, 2, 40, 64, seed=1), _rand(2, 2, 40, 64, seed=2)
    tree = ops.draft_tree(_i32([[-1, 0, 1]] * 2))
    a = ops.tree_attention(qkv, kc, vc, _i32([1000, -5]), tree, 4, _i32([-9, -1]))
    b = ops.tree_attention(qkv, kc, vc, _i32([40, 0]), tree, 4)
    assert torch.equal(a, b)
    c = ops.tree_attention(qkv, kc, vc, _i32([40, 40]), tree, 4, _i32([100, 40]))  # starts behind the end: no context
    assert torch.equal(c, ops.tree_attention(qkv, kc, vc, _i32([0, 0]), tree, 4))


@pytest.mark.parametrize("Hq,Hkv,D,slots", [(8, 2, 128, 2000), (8, 2, 128, 60), (3, 1, 32, 60)])
def test_attention_of_masks_with_holes(Hq, Hkv, D, slots):
    """a plan of the caller's own: nodes that see nothing between others, and nodes that see others than ancestors"""
    N = 12
    see = [1, 0, 0b101, 0, 0, 0b100100, 1 << 6, 0, 0b111111000001 & 0b000100000001, 0, 0b10000000101, 0]
    see = [s if s == 0 else s | 1 << i for i, s in enumerate(see)]
    qkv, kc, vc = _rand(N, (Hq + 2 * Hkv) * D, seed=1), _rand(1, Hkv, slots, D, seed=2), _rand(1, Hkv, slots, D, seed=3)
    tree = ops.DraftTree(_i32([[-1] * N]), torch.tensor([see], device=DEV), _i32([[0] * N]))
    o = ops.tree_attention(qkv, kc, vc, _i32([slots]), tree, Hq)
    want = ops.tree_attention(qkv.cpu().double(), kc.cpu().double(), vc.cpu().double(), torch.tensor([slots], dtype=torch.int32),
                              ops.DraftTree(*(t.cpu() for t in (tree.parent, tree.see, tree.pos))), Hq)
    assert (o[[i for i, s in enumerate(see) if not s]] == 0).all()
    # two roundings of half a step, of p in a mean of |v| below 1 and of the output below 2 here, and scores as in _attention
    assert ((o.cpu().double() - want).abs() <= 2 ** -8 * (1 + want.abs()) + 2 * 2 ** -24 * (16 * D + slots)).all()


def test_attention_gives_a_row_the_same_beside_others():
    """a row's bits do not depend on the other rows of the batch, nor a node's on the nodes that it does not see"""
    B, N, Hq, Hkv, D = 3, 10, 8, 2, 128
    qkv, kc, vc = _rand(B * N, (Hq + 2 * Hkv) * D), _rand(B, Hkv, 500, D, seed=1), _rand(B, Hkv, 500, D, seed=2)
    lens, parents = [490, 3, 200], plain.trees(B, N, 0)
    a = ops.tree_attention(qkv, kc, vc, _i32(lens), ops.draft_tree(_i32(parents)), Hq)
    others = qkv.clone()
    others[N:] *= 30  # the other rows' queries and keys
    others[N - 1] *= 30  # the last node of row 0: nobody's ancestor
    b = ops.tree_attention(others, kc, vc, _i32([490, 400, 1]), ops.draft_tree(_i32(parents)), Hq)
    assert torch.equal(a[:N - 1], b[:N - 1])


def test_attention_nothing_to_do():
    tree = ops.draft_tree(torch.zeros(0, 3, dtype=torch.int32, device=DEV))
    o = ops.tree_attention(torch.zeros(0, 512, dtype=BF16, device=DEV), *(torch.zeros(0, 2, 9, 64, dtype=BF16, device=DEV) for _ in "kv"), _i32([]), tree, 4)
    assert o.shape == (0, 256)


def test_attention_offsets_past_32_bits():
    """a cache of more than 2^32 bytes and 2^31 elements: the last row's keys lie behind both"""
    B, Hkv, D, slots = 9, 8, 128, 262144  # 2.4 G elements, 4.8 GB each
    kc, vc = (torch.zeros(B, Hkv, slots, D, dtype=BF16, device=DEV) for _ in "kv")
    lens, N = [5] * (B - 1) + [slots], 2
    kc[-1, -1, -300:], vc[-1, -1, -300:] = _rand(300, D, seed=1), _rand(300, D, seed=2)
    qkv = _rand(B * N, (8 + 2 * Hkv) * D)
    starts = [0] * (B - 1) + [slots - 300]
    parents = [[-1, 0]] * B
    o = ops.tree_attention(qkv, kc, vc, _i32(lens), ops.draft_tree(_i32(parents)), 8, _i32(starts))
    small = ops.tree_attention(qkv[-N:], kc[-1:, :, -300:].contiguous(), vc[-1:, :, -300:].contiguous(), _i32([300]),
                               ops.draft_tree(_i32(parents[:1])), 8)
    assert torch.allclose(o[-N:].float(), small.float(), rtol=2 ** -6, atol=2 ** -8)  # two roundings of p and of o, other partitions


# ------------------------------------------------------------------------------------------ acceptance
@pytest.mark.parametrize("dtype,D,extra", [(BF16, 128, 0), (BF16, 64, 3), (F32, 20, 0), (BF16, 6, 0)])
@pytest.mark.parametrize("N", [1, 6, 64])
def test_accept(dtype, D, extra, N):
    r = random.Random(N)
    B, L, Hq, Hkv, slots = 7, 3, 4, 2, 90
    parents, counts = plain.trees(B, N, N, 3), [r.randint(0, N) for _ in range(B)]
    parents[0], counts[0] = [-1] + list(range(N - 1)), N  # a chain that is accepted whole
    tokens, choice = ([[r.randrange(3) + 2 ** 40 for _ in range(N)] for _ in range(B)] for _ in "tc")
    choice[0] = tokens[0][1:] + [9]
    lens = [r.randint(0, slots) for _ in range(B - 1)] + [slots + 5]
    lens[0] = 20
    rows = [_rand(B * N, (Hq + 2 * Hkv) * D + extra, dtype=dtype, seed=i) for i in range(L)]
    drafts = [x[:, :(Hq + 2 * Hkv) * D] for x in rows]
    whole = [_rand(L, B + 1, Hkv, slots, D, dtype=dtype, seed=9 + i) for i in range(2)]
    kc, vc = (c[:, :B] for c in whole)  # the first rows of a larger cache
    cpu = [c[:, :B].cpu().contiguous() for c in whole]
    rest = [c[:, B:].clone() for c in whole]
    t = lambda x: torch.tensor(x)
    want = ops.tree_accept(ops.draft_tree(t(parents).int(), t(counts).int()), t(tokens), t(choice), [x.cpu() for x in drafts], *cpu, t(lens).int())
    got = ops.tree_accept(ops.draft_tree(_i32(parents), _i32(counts)), t(tokens).to(DEV), t(choice).to(DEV), drafts, kc, vc, _i32(lens))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(kc.cpu(), cpu[0]) and torch.equal(vc.cpu(), cpu[1])
    assert all(torch.equal(c[:, B:], r0) for c, r0 in zip(whole, rest))


# ------------------------------------------------------------------------------------------ alternatives
def _check_alternatives(x, t, top, c, grad=True):
    T, V = x.shape
    x = x.detach().requires_grad_(grad)
    lp, ent, tl, ids = ops.token_alternatives(x, t, top, c)
    wlp, went, wtl, wids, ez, zt, ls = plain.alternatives(x, t, top, c)
    assert torch.equal(ids.cpu(), wids)
    # fp32: the chain of sums (2^-24 each; a thread's V / 256 values at most and 16 joints, doubled for the entropy's), z of three roundings, exp
    # and log of their argument's rounding and two steps
    unit = 2 ** -23 * (V / 256 + 24 + 2 * ls.abs() + 2 * ez)
    for got, want, tol in ((lp, wlp, unit + 2 ** -22 * zt), (ent, went, unit * (2 + ez)),
                           (tl, wtl, unit[:, None] + 2 ** -22 * (wtl.abs() + ls.abs()[:, None]))):
        got = got.detach().cpu().double()
        ok = (got == want) | ((got - want).abs() <= tol) | (torch.isnan(got) & torch.isnan(want))
        assert ok.all(), ((got - want).abs() / tol)[~ok].max()
    if not grad:
        return
    g = [_rand(T, dtype=F32, seed=1), _rand(T, dtype=F32, seed=2), _rand(T, top, dtype=F32, seed=3)]
    d, = torch.autograd.grad([lp, ent, tl], x, g)
    assert d.dtype == x.dtype and d.shape == x.shape
    tt = t if t is not None else torch.full((T,), -1)
    want, size = plain.gradient(x, tt, ids, c, *g)
    # the stored value's rounding, and each term's error in fp32: p's is that of its exponent
    tol = (torch.finfo(x.dtype).eps / 2 if x.dtype == BF16 else 2 ** -23) * want.abs() + (3 * unit[:, None] + 2 ** -20) * size + 1e-37
    live = torch.isfinite(want).all(1)  # rows of -inf alone have no formula: no gradient
    err = (d.cpu().double() - want).abs()
    assert (err[live] <= tol[live]).all(), (err / tol)[live].max()
    assert (d[~live.to(DEV)] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (3, 7, 7), (5, 33, 32), (9, 512, 20), (4, 1000, 1), (17, 1003, 8), (3, 30522, 32), (2, 32002, 20),
                                     (2, 50272, 5), (1, 131072, 8), (1, 151937, 8)])
def test_alternatives(T, V, top, dtype):
    t = torch.randint(-2, V, (T,), generator=torch.Generator().manual_seed(T)).to(DEV)
    t[0] = V - 1
    _check_alternatives(_rand(T, V, dtype=dtype, seed=V) * 3, t, top, 1 / 0.7)


def test_alternatives_of_many_rows():
    x = _rand(700, 2048, seed=1) * 2
    _check_alternatives(x, torch.randint(0, 2048, (700,)).to(DEV), 10, 1.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [40, 1030, 32000])
def test_alternatives_of_rows_with_a_pattern(V, dtype):
    """equal values, sorted ones, the best ones far apart and in one thread's or one wave's share, few that are left by a mask"""
    i = torch.arange(V, device=DEV).float()
    x = torch.stack([0 * i, i / V, -i / V, (i % 8), (i % 64 == 5) * 3.0 - i / V, (i // 8 % 64 == 3) * 9.0 + i / V, (i // 8 % 256 == 7) * 9.0 - i / V,
                     (i // 8 % 1024 == 2) * 9.0, -1000 * (i != V - 1), 100 + i % 3, -0.0 * (i % 2)])
    masked = torch.full((7, V), -math.inf, device=DEV)
    masked[0, V - 1], masked[1, 0], masked[2, ::9], masked[3, V // 2:], masked[4, 3], masked[4, 5] = 1, 2, 0.5, 0.25, 1, 1
    masked[6] = torch.finfo(dtype).min
    x = torch.cat([x, masked]).to(dtype)
    t = torch.zeros(len(x), dtype=torch.long, device=DEV)
    for top in (1, 8, 20, 32):
        _check_alternatives(x, t, top, 1 / 0.7, grad=top == 8)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [9000, 32002, 50272, 70001, 140001])
def test_alternatives_of_many_rows_are_those_of_few(V, dtype):
    """more rows than CUs take other forms than a few do; random rows, and rows whose best lie in one thread's or one wave's share"""
    i = torch.arange(V, device=DEV).float()
    x = torch.cat([_rand(20, V, dtype=F32, seed=V) * 3, torch.stack([0 * i, i / V, (i // 8 % 256 == 7) * 9.0 - i / V, (i // 4 % 512 == 9) * 9.0 + i / V,
                                                                     (i // 8 % 1024 == 2) * 9.0, torch.where(i == V - 2, 1.0, -math.inf)])]).to(dtype)
    t = torch.arange(len(x), device=DEV)
    few = ops.token_alternatives(x, t, 20, 1 / 0.7)
    many = ops.token_alternatives(x.repeat(14, 1), t.repeat(14), 20, 1 / 0.7)
    assert torch.equal(many[3], few[3].repeat(14, 1))
    for a, b in zip(many[:3], few):  # other orders of the sums: 2^-23 (V / 256 + 16) each, of values below 16, and twice that of E|z|
        b = b.repeat(14, *[1] * (b.dim() - 1))
        assert ((a == b) | ((a - b).abs() <= 16 * 2 ** -23 * (V / 256 + 16))).all()


def test_alternatives_of_rows_that_are_no_numbers():
    x = _rand(4, 600, seed=1)
    x[0, 300], x[1, :], x[2, 17], x[3, 599] = math.nan, math.nan, math.inf, math.nan
    x.requires_grad_(True)
    lp, ent, top, ids = ops.token_alternatives(x, torch.tensor([0, 1, 2, -1], device=DEV), 4)
    assert torch.isnan(lp[:3]).all() and lp[3] == 0 and torch.isnan(ent).all() and torch.isnan(top).all()
    want = plain.alternatives(x, None, 4, 1.0)[3]
    assert torch.equal(ids.cpu(), want) and ids[2, 0] == 17
    lp.sum().backward()
    assert torch.isnan(x.grad[:3]).any(1).all()


def test_alternatives_of_a_target_outside():
    x = _rand(3, 100, seed=1)
    lp, ent, top, ids = ops.token_alternatives(x, torch.tensor([100, 2 ** 40, -2 ** 40], device=DEV), 2)
    assert torch.isnan(lp[:2]).all() and lp[2] == 0 and torch.isfinite(ent).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pitch,at", [(1011, 0), (1011, 3), (1024, 8), (1024, 1)])
def test_alternatives_of_strided_rows(pitch, at, dtype):
    wide = _rand(6, pitch, dtype=dtype, seed=2)
    x = wide[:, at:at + 1000]
    a = ops.token_alternatives(x, None, 9)
    b = ops.token_alternatives(x.contiguous(), None, 9)
    assert torch.equal(a[3], b[3])
    _check_alternatives(x, torch.arange(6, device=DEV), 9, 1.0)
    _check_alternatives(wide.t()[:6].t().contiguous().t()[:, :6], torch.zeros(6, dtype=torch.int32, device=DEV), 2, 1.0)


def test_alternatives_without_targets():
    _check_alternatives(_rand(5, 300, dtype=F32, seed=1), None, 7, 1.0)


def test_alternatives_offsets_past_32_bits():
    """rows 2^30 + 5 elements apart: the last one lies behind 2^31 elements and 2^32 bytes"""
    V, pitch = 1000, 2 ** 30 + 5
    store = torch.empty(2 * pitch + V, dtype=BF16, device=DEV)
    x = store.as_strided((3, V), (pitch, 1))
    x.copy_(_rand(3, V, seed=1))
    _check_alternatives(x, torch.tensor([0, 999, 500], device=DEV), 5, 1.0)


def test_alternatives_nothing_to_do():
    x = torch.zeros(0, 100, dtype=BF16, device=DEV, requires_grad=True)
    lp, ent, top, ids = ops.token_alternatives(x, torch.zeros(0, dtype=torch.long, device=DEV), 3)
    assert lp.shape == ent.shape == (0,) and top.shape == ids.shape == (0, 3)
    lp.sum().backward()
    assert x.grad.shape == (0, 100)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_alternatives_gradient_of_one_output(which):
    x = _rand(5, 700, dtype=F32, seed=3).requires_grad_(True)
    t = torch.tensor([0, 699, -1, 5, 5], device=DEV)
    out = ops.token_alternatives(x, t, 6, 0.9)
    out[which].sum().backward()
    gs = [torch.ones_like(o) if i == which else torch.zeros_like(o) for i, o in enumerate(out[:3])]
    want, size = plain.gradient(x, t, out[3], 0.9, *(g.detach() for g in gs))
    assert ((x.grad.cpu().double() - want).abs() <= 2 ** -17 * size + 1e-30).all()  # as above: 2^-23 (3 + 24 + 2 log 700 + ...) of the terms


def test_alternatives_gradient_against_differences():
    x = _rand(3, 50, dtype=F32, seed=4)
    u = _rand(3, 50, dtype=F32, seed=5)
    t = torch.tensor([1, 49, 7], device=DEV)

    def f(y):
        lp, ent, top, _ = ops.token_alternatives(y, t, 4, 1.2)
        return (lp.double().sum() + 0.5 * ent.double().sum() - 0.3 * top.double().sum())

    y = x.clone().requires_grad_(True)
    f(y).backward()
    h = 2 ** -6
    diff = (f(x + h * u) - f(x - h * u)) / (2 * h)
    # differences: h^2 / 6 of the third derivative (under 100 for these three rows), 18 values of 2^-20 over 2 h
    assert abs((y.grad.double() * u.double()).sum() - diff) <= h * h / 6 * 100 + 18 * 2 ** -20 / (2 * h)


# ------------------------------------------------------------------------------------------ how they are called
def _step(qkv, kc, vc, k_all, v_all, parents, counts, lens, tokens, targets):
    """one checked step over a single layer: plan, attention, logits, alternatives, acceptance"""
    B, N = parents.shape
    tree = ops.draft_tree(parents, counts, lens)
    o = ops.tree_attention(qkv, kc, vc, lens, tree, 8)
    lp, ent, top, ids = ops.token_alternatives(o[:, :7], targets, 4)  # a vocabulary of 7, in place of a head's product
    return (o, lp, ent, top, ids, *ops.tree_accept(tree, tokens, ids[:, 0].view(B, N).contiguous(), [qkv], k_all, v_all, lens))


def _step_inputs(seed, B=3, N=12, slots=400):
    k_all, v_all = _rand(1, B, 2, slots, 64, seed=seed + 1), _rand(1, B, 2, slots, 64, seed=seed + 2)
    tokens = torch.randint(0, 7, (B, N), generator=torch.Generator().manual_seed(seed)).to(DEV)
    return [_rand(B * N, 12 * 64, seed=seed), k_all[0], v_all[0], k_all, v_all, _i32(plain.trees(B, N, seed)), _i32([N, N - 3, 0]),
            _i32([380, 37, 5]), tokens, torch.randint(-1, 7, (B * N,), generator=torch.Generator().manual_seed(seed)).to(DEV)]


def test_a_captured_step_replays():
    """replays over new contents, with the eager step in between, give the eager results"""
    s = _step_inputs(0)
    work = [t.clone() for t in s]
    work[1], work[2] = work[3][0], work[4][0]  # the layer's cache is a view of the whole one
    held = {}
    runner = GraphRunner()
    runner.capture(lambda: held.update(out=_step(*work)), "step")
    for seed in (10, 20, 30):
        new = _step_inputs(seed)
        for a, b in zip(work, new):
            a.copy_(b)
        runner.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held["out"]] + [work[3].clone(), work[4].clone()]
        want = list(_step(*new)) + [new[3], new[4]]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_captured_steps_replay_at_once():
    """each with memory of its own, on two streams"""
    runs = []
    for seed in (0, 50):
        s, graph = _step_inputs(seed), torch.cuda.CUDAGraph()
        _step(*s)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = _step(*s)
        runs.append((out, graph, s))
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        for (_, graph, _), st in zip(runs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for seed, (out, _, _) in zip((0, 50), runs):
        for a, b in zip(out, _step(*_step_inputs(seed))):
            assert torch.equal(a, b)


def test_steps_on_two_streams_at_once():
    inputs = [_step_inputs(seed, B=3) for seed in (0, 70)]
    want = [_step(*_step_inputs(seed, B=3)) for seed in (0, 70)]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_step(*inputs[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for out in runs:
            for a, b in zip(out, w):
                assert torch.equal(a, b)


def test_a_captured_gradient_replays():
    x, t = _rand(9, 1003, dtype=F32, seed=1), torch.arange(-1, 8, device=DEV)
    g = [_rand(9, dtype=F32, seed=2), _rand(9, dtype=F32, seed=3), _rand(9, 5, dtype=F32, seed=4)]

    def step(x):
        y = x.detach().requires_grad_(True)
        lp, ent, top, ids = ops.token_alternatives(y, t, 5, 1.1)
        return lp.detach(), ent.detach(), top.detach(), ids, torch.autograd.grad([lp, ent, top], y, g)[0]

    held, runner, work = {}, GraphRunner(), x.clone()
    runner.capture(lambda: held.update(out=step(work)), "step")
    for seed in (1, 5, 6):
        new = _rand(9, 1003, dtype=F32, seed=seed)
        work.copy_(new)
        runner.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in held["out"]]
        for a, b in zip(got, step(new)):
            assert torch.equal(a, b)


def test_no_second_derivative():
    x = _rand(2, 50, dtype=F32).requires_grad_(True)
    lp = ops.token_alternatives(x, torch.tensor([1, 2], device=DEV), 2)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(lp.sum(), x, create_graph=True)


def test_runs_repeat_bit_by_bit():
    qkv, kc, vc = _rand(8 * 20, 12 * 128, seed=1), _rand(8, 2, 3000, 128, seed=2), _rand(8, 2, 3000, 128, seed=3)
    tree, lens = ops.draft_tree(_i32(plain.trees(8, 20, 0))), _i32([3000, 1, 700, 0, 64, 2999, 1500, 33])
    x = _rand(40, 32000, seed=4).requires_grad_(True)
    first = None
    for _ in range(4):
        lp, ent, top, ids = ops.token_alternatives(x, torch.arange(40, device=DEV), 20)
        out = [ops.tree_attention(qkv, kc, vc, lens, tree, 8), lp, ent, top, ids, torch.autograd.grad(lp.sum() + ent.sum() + top.sum(), x)[0]]
        first = first or out
        for a, b in zip(out, first):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [
    lambda: ops.draft_tree(_i32([[-1, 0]]), nodes=torch.tensor([2], dtype=torch.int32)),
    lambda: ops.tree_attention(_rand(2, 512), _rand(1, 2, 9, 64), _rand(1, 2, 9, 64).cpu(), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4),
    lambda: ops.tree_attention(_rand(2, 512), _rand(1, 2, 9, 64), _rand(1, 2, 9, 128)[..., :64], _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4),
    lambda: ops.tree_attention(_rand(2, 512), _rand(1, 2, 9, 64), _rand(1, 2, 9, 64), _i32([3]), ops.draft_tree(torch.tensor([[-1, 0]], dtype=torch.int32)), 4),
    lambda: ops.tree_attention(_rand(2, 512).half(), *(_rand(1, 2, 9, 64).half() for _ in "kv"), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4),
    lambda: ops.tree_attention(_rand(2, 512), _rand(1, 2, 9, 64), _rand(1, 2, 9, 64), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4,
                               out=torch.empty(2, 255, dtype=BF16, device=DEV)),
    lambda: ops.tree_accept(ops.draft_tree(_i32([[-1, 0]])), *(torch.zeros(1, 2, dtype=torch.long, device=DEV) for _ in "tc"), [_rand(2, 512)],
                            _rand(1, 1, 2, 9, 64), _rand(1, 1, 2, 64, 9).transpose(3, 4), _i32([3])),
    lambda: ops.tree_attention(_rand(2, 512).requires_grad_(True), _rand(1, 2, 9, 64), _rand(1, 2, 9, 64), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4),
    lambda: ops.tree_attention(_rand(2, 512), _rand(1, 2, 9, 64), _rand(1, 2, 9, 64), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4, scale=-1.0),
    lambda: ops.tree_attention(_rand(2, 512), *(torch.zeros(1, 2, 9, 64, dtype=torch.uint8, device=DEV) for _ in "kv"), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4),
    lambda: ops.draft_tree(torch.zeros(2, 65, dtype=torch.int32, device=DEV)),
    lambda: ops.tree_attention(_rand(2, 512), _rand(1, 2, 9, 64), _rand(1, 2, 9, 64), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4,
                               out=torch.empty(1, 256, dtype=BF16, device=DEV).expand(2, 256)),
    lambda: _in_place(_rand(2, 512)),
    lambda: _over_the_cache(_rand(1, 2, 9, 64)),
    lambda: ops.tree_attention(_rand(0, 512), _rand(2, 2, 9, 64), _rand(2, 2, 9, 64), _i32([3, 3]), _empty(2, 0), 4),
    lambda: ops.tree_attention(_rand(130, 512), _rand(2, 2, 9, 64), _rand(2, 2, 9, 64), _i32([3, 3]), _empty(2, 65), 4),
    lambda: ops.tree_accept(_empty(2, 0), *(torch.zeros(2, 0, dtype=torch.long, device=DEV) for _ in "tc"), [_rand(0, 512)],
                            *(_rand(1, 2, 2, 9, 64) for _ in "kv"), _i32([3, 3])),
    lambda: ops.tree_accept(ops.draft_tree(_i32([[-1, 0]])), *(torch.zeros(1, 2, dtype=torch.long, device=DEV) for _ in "tc"), [_rand(2, 512)],
                            *[_rand(1, 1, 2, 9, 64)] * 2, _i32([3])),
    lambda: ops.token_alternatives(_rand(1, 1).expand(1 << 22, 1), None, 1),
    lambda: ops.tree_attention(_rand(2, 512, dtype=F32), *(torch.zeros(1, 1, 9, 128, dtype=torch.uint8, device=DEV) for _ in "kv"), _i32([3]),
                               ops.draft_tree(_i32([[-1, 0]])), 2, k_scale=torch.ones(1, 1, 9, device=DEV), v_scale=torch.ones(1, 1, 9, device=DEV)),
    lambda: ops.tree_attention(_rand(2, 512), *(torch.zeros(1, 1, 9, 128, dtype=torch.uint8, device=DEV) for _ in "kv"), _i32([3]),
                               ops.draft_tree(_i32([[-1, 0]])), 2, k_scale=torch.ones(1, 1, 8, device=DEV), v_scale=torch.ones(1, 1, 8, device=DEV)),
    lambda: ops.tree_attention(_rand(2, 512), *(_rand(1, 1, 9, 128) for _ in "kv"), _i32([3]),
                               ops.draft_tree(_i32([[-1, 0]])), 2, k_scale=torch.ones(1, 1, 9, device=DEV), v_scale=torch.ones(1, 1, 9, device=DEV)),
    lambda: ops.tree_accept(ops.draft_tree(_i32([[-1, 0]])), *(torch.zeros(1, 2, dtype=torch.long, device=DEV) for _ in "tc"), [_rand(2, 512)],
                            *(torch.zeros(1, 1, 2, 9, 0, dtype=BF16, device=DEV) for _ in "kv"), _i32([3])),
    lambda: ops.token_alternatives(_rand(2, 50), None, 33),
    lambda: ops.token_alternatives(_rand(2, 50), None, 2, 1e-60),
    lambda: ops.token_alternatives(_rand(2, 50), None, 2, math.inf),
    lambda: ops.token_alternatives(_rand(2, 50), torch.zeros(3, dtype=torch.long, device=DEV), 2),
    lambda: ops.token_alternatives(_rand(2, 50).half(), None, 2),
    lambda: ops.token_alternatives(_rand(2, 50), torch.zeros(2, dtype=torch.long), 2),
])
def test_refused(bad):
    with pytest.raises((ValueError, RuntimeError)):
        bad()


def _empty(*shape):
    return ops.DraftTree(*(torch.zeros(*shape, dtype=t, device=DEV) for t in (torch.int32, torch.int64, torch.int32)))


def _over_the_cache(kc):
    return ops.tree_attention(_rand(2, 512), kc, _rand(1, 2, 9, 64), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4, out=kc.view(-1)[:512].view(2, 256))


def _in_place(qkv):
    return ops.tree_attention(qkv, _rand(1, 2, 9, 64), _rand(1, 2, 9, 64), _i32([3]), ops.draft_tree(_i32([[-1, 0]])), 4, out=qkv[:, :256])


@pytest.mark.parametrize("preset", ["tiny-mistral", "tiny-opt"])
def test_verify_of_idle_rows_and_of_trees_past_the_last_position(preset):
    """an idle row's next token is -1; nodes past the model's positions leave those before them as they are"""
    cfg = models.resolve_preset(preset)
    m = models.CausalLM(cfg, device=DEV, dtype=BF16, seed=3)
    B, N, S = 3, 6, cfg.max_position
    cache = KVCache(cfg.num_layers, B, cfg.num_kv_heads, S, cfg.head_dim, DEV)
    cache.k.normal_(), cache.v.normal_()
    kv_len = _i32([9, 0, S - 3])
    chain, tokens = _i32([[-1] + list(range(N - 1))] * B), torch.arange(3, 3 + B * N, device=DEV).view(B, N)
    idle = tokens.clone()
    idle[1] = -1
    h = m.verify(idle, ops.draft_tree(chain, _i32([N, 0, N]), kv_len), kv_len, None, cache)[0].view(B, N, -1)
    want = m.verify(tokens, ops.draft_tree(chain, _i32([N, 0, 3]), kv_len), kv_len, None, cache)[0].view(B, N, -1)
    assert torch.equal(h[0], want[0])
    # six nodes leave the context's last 61 keys of 64 to a stage of their own where three take them into theirs: p is rounded to bf16 against
    # another maximum, so the states are apart by roundings of half a step, 16 on their way through two layers as below
    x, y = h[2, :3].float(), want[2, :3].float()
    assert (x - y).pow(2).mean().sqrt() <= 16 ** 0.5 * 2 ** -8 * y.pow(2).mean().sqrt()


def test_a_model_checks_drafts_like_single_steps():
    """hidden states of a chain of drafts and those of decoding it token by token, in bf16"""
    cfg = models.resolve_preset("tiny-mistral")
    m = models.CausalLM(cfg, device=DEV, dtype=BF16, seed=1)
    B, S, N, slots = 2, 90, 6, 128
    ids = torch.randint(3, 500, (B, S), generator=torch.Generator().manual_seed(0)).to(DEV)
    start, kv_len = _i32([0, 31]), _i32([S, S])
    a, b = (KVCache(cfg.num_layers, B, cfg.num_kv_heads, slots, cfg.head_dim, DEV) for _ in "ab")
    m.prefill(ids, start, a)
    m.prefill(ids, start, b)
    tokens = torch.randint(3, 500, (B, N), generator=torch.Generator().manual_seed(1)).to(DEV)
    tree = ops.draft_tree(_i32([[-1] + list(range(N - 1))] * B), pos0=kv_len - start)
    h, drafts = m.verify(tokens, tree, kv_len, start, a)
    choice = torch.cat([tokens[:, 1:], tokens[:, :1]], 1)  # agrees with all of them
    count, path, after = ops.tree_accept(tree, tokens, choice, drafts, a.k, a.v, kv_len)
    assert count.tolist() == [N, N] and path.tolist() == [list(range(N))] * B and torch.equal(after, tokens[:, 0])
    single = torch.stack([m.decode(tokens[:, i], kv_len - start + i, kv_len + i, kv_len + i + 1, start, b) for i in range(N)], 1)
    x, y = h.view(B, N, -1).float(), single.float()
    # normalised states (of size 1), each of about 16 roundings to bf16 on its way through two layers
    assert ((x - y).pow(2).mean().sqrt() <= 16 ** 0.5 * 2 ** -8 * y.pow(2).mean().sqrt())
    for c, d in ((a.k, b.k), (a.v, b.v)):
        c, d = c[:, :, :, S:S + N].float(), d[:, :, :, S:S + N].float()
        assert (c - d).pow(2).mean().sqrt() <= 16 ** 0.5 * 2 ** -8 * d.pow(2).mean().sqrt()
