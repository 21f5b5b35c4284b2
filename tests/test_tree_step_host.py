"""CPU checks of a tree-drafted step's entries: argument checks of the C ABI and of the wrappers (no kernel is launched),
registered schemas, the static check of the tree attention's LDS waits, the oracle against itself."""
import ctypes
import random

import pytest
import torch

import tree_step_ref as R
from test_lds_waits import _asm, asm_lds


def refused(lib, rc, text):
    return rc == 1 and text in lib.dsa_last_error_message()


def test_plan_c_checks(dsa):
    lib = dsa.load_library()

    def call(new=16, table=16, free=16, count=16, par=None, B=4, T=8, mb=4, bs=16, room=8, W=1, win=-1, cu=16, pos=16,
             mask=16):
        return lib.dsa_paged_plan(new, 16, table, free, count, par, B, T, mb, bs, room, W, win, cu, 16, pos, 16, 16, mask,
                                  None)

    for kw, msg in [(dict(B=0), b"B must"), (dict(B=16385), b"B must"), (dict(bs=0), b"page"), (dict(mb=0), b"page"),
                    (dict(mb=2**30), b"page"), (dict(room=-1), b"page"), (dict(room=2**31), b"page"),
                    (dict(T=-1), b"T must"), (dict(T=2**30), b"T must"), (dict(par=16, W=-1), b"mask_words"),
                    (dict(par=16, T=2**22 + 1), b"2^22 with parents"),
                    (dict(par=16, W=65), b"mask_words"), (dict(win=-2), b"win_left"), (dict(new=None), b"null"),
                    (dict(table=None), b"null"), (dict(free=None), b"null"), (dict(count=None), b"null"),
                    (dict(cu=None), b"null"), (dict(pos=None), b"null"), (dict(par=16, mask=None), b"null")]:
        assert refused(lib, call(**kw), msg), kw


def test_free_c_checks(dsa):
    lib = dsa.load_library()
    call = lambda keep=16, free=16, B=4, mb=4, bs=16, room=8: lib.dsa_paged_free(keep, 16, free, 16, B, mb, bs, room, None)
    for kw, msg in [(dict(B=0), b"B must"), (dict(B=16385), b"B must"), (dict(bs=0), b"page"), (dict(mb=0), b"page"),
                    (dict(keep=None), b"null"), (dict(free=None), b"null")]:
        assert refused(lib, call(**kw), msg), kw


def test_tree_attention_c_checks(dsa):
    lib = dsa.load_library()

    def call(kind=1, q=16, mask=16, W=1, pos=None, T=4, B=2, S=2, H=8, G=2, D=64, nb=4, bs=16, mb=2, win=-1, scale=1.0,
             ws=16, nws=1 << 30, cu=None):
        return lib.dsa_paged_tree_fwd(kind, q, 16, 16, 16, mask, W, pos, cu, None, 16, T, B, S, H, G, D, nb, bs, mb, win,
                                      None, scale, 16, 16, ws, nws, None)

    for kw, msg in [(dict(kind=0), b"kind"), (dict(D=96), b"D must"), (dict(H=7), b"multiple of kv_group"),
                    (dict(bs=0), b"page"), (dict(mb=2**27), b"range"), (dict(T=5), b"B * S"), (dict(win=-2), b"win_left"),
                    (dict(scale=0.0), b"sm_scale"), (dict(q=None), b"null"), (dict(q=18), b"16 bytes"),
                    (dict(W=0), b"mask_words"), (dict(W=65), b"mask_words"), (dict(mask=None), b"null"),
                    (dict(mask=20), b"8 bytes"), (dict(win=3), b"null"), (dict(T=200, S=100), b"64 * mask_words"),
                    (dict(nws=0), b"workspace"), (dict(ws=None), b"workspace")]:
        assert refused(lib, call(**kw), msg), kw
    assert call(T=0, S=0) == 0
    assert lib.dsa_paged_tree_workspace_size(8, 1, 64, 4, 128, 4160) > 0
    assert lib.dsa_paged_tree_workspace_size(0, 1, 64, 4, 128, 4160) == 0
    assert lib.dsa_paged_tree_workspace_size(8, 1, 64, 3, 128, 4160) == 0


def test_accept_c_checks(dsa):
    lib = dsa.load_library()

    def call(kind=1, x=16, stride=100, T=4, V=100, tok=16, cu=16, B=2, P=3, ws=16, n=1 << 30):
        return lib.dsa_tree_accept(kind, x, stride, T, V, tok, 16, cu, B, P, 16, 16, 16, ws, n, None)

    for kw, msg in [(dict(kind=0), b"kind"), (dict(T=-1), b"T must"), (dict(T=2**30), b"T must"), (dict(V=0), b"V must"),
                    (dict(V=2**30), b"V must"), (dict(B=0), b"bad B"), (dict(B=65536), b"bad B"), (dict(P=0), b"max_path"),
                    (dict(P=2**31), b"max_path"), (dict(x=None), b"null"), (dict(tok=None), b"null"),
                    (dict(cu=None), b"null"), (dict(x=17), b"element"), (dict(kind=3, x=18), b"element"),
                    (dict(stride=99), b"overlap"), (dict(stride=2**59), b"row_stride"), (dict(n=0), b"workspace"),
                    (dict(ws=None), b"workspace"), (dict(ws=20), b"workspace")]:
        assert refused(lib, call(**kw), msg), kw
    assert lib.dsa_tree_accept_workspace_size(5, 4, 0) == 0
    assert lib.dsa_tree_accept_workspace_size(1, 0, 100) == 0


def test_commit_c_checks(dsa):
    lib = dsa.load_library()

    def call(at=(4096, 1 << 20), rows=(64, 64), table=16, B=2, P=3, nb=4, bs=16, mb=2, n=None):
        n = len(at) if n is None else n
        return lib.dsa_paged_commit((ctypes.c_void_p * len(at))(*at), (ctypes.c_int64 * len(rows))(*rows), n, table, 16, 16,
                                    16, B, P, nb, bs, mb, None)

    for kw, msg in [(dict(n=-1), b"number"), (dict(n=65537), b"number"), (dict(B=0), b"bad B"), (dict(B=65536), b"bad B"),
                    (dict(P=-1), b"max_path"), (dict(bs=0), b"page"), (dict(nb=0), b"page"), (dict(nb=2**31), b"page"),
                    (dict(mb=0), b"page"), (dict(table=None), b"null"), (dict(at=(None, 4096)), b"null cache"),
                    (dict(rows=(6, 64)), b"multiples of 4"), (dict(rows=(0, 64)), b"multiples of 4"),
                    (dict(at=(4098, 1 << 20)), b"multiples of 4"), (dict(rows=(1 << 23, 64)), b"multiples of 4"),
                    (dict(at=(4096, 4096)), b"overlap"), (dict(at=(1 << 20, (1 << 20) - 4)), b"overlap"),
                    (dict(at=tuple(1 << 40 | i << 30 for i in range(64)), rows=(1 << 22,) * 64, B=65535, nb=1, bs=1),
                     b"range")]:
        assert refused(lib, call(**kw), msg), kw
    assert call(P=0) == 0 and call(n=0) == 0


def test_host_tensors_are_refused(dsa):
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP"):
        dsa.paged_plan(i, i, i.view(4, 1), i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="HIP"):
        dsa.paged_free(i, i.view(4, 1), i, i[:1], 16)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    m = torch.zeros(4, 1, dtype=torch.int64)
    with pytest.raises(ValueError, match="HIP"):
        dsa.paged_tree_fwd(q, c, c, i.view(1, 4), m, actual_seq_lengths_query=i[:1], actual_seq_lengths_kv=i[:1])
    with pytest.raises(ValueError, match="HIP"):
        dsa.tree_accept(torch.zeros(4, 8), i, i, actual_seq_lengths_query=i[:1], max_path=2)
    with pytest.raises(ValueError, match="HIP"):
        dsa.paged_commit(c, i.view(1, 4), i[:1], i.view(1, 4), i[:1])


def test_wrappers_name_what_they_refuse(dsa):
    i = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    m = torch.zeros(4, 1, dtype=torch.int64)
    tree = lambda mask=m, **kw: dsa.paged_tree_fwd(q, c, c, i.view(1, 4), mask, actual_seq_lengths_query=i[:1],
                                                   actual_seq_lengths_kv=i[:1], **kw)
    for mask in (m.int(), m.view(1, 4), m.view(-1), torch.zeros(5, 1, dtype=torch.int64), torch.zeros(4, 1)):
        with pytest.raises(ValueError, match="tree_mask must be"):
            tree(mask)
    with pytest.raises(ValueError, match="1 to 64 words"):
        tree(torch.zeros(4, 65, dtype=torch.int64))
    with pytest.raises(ValueError, match="positions"):
        tree(win_left=3)
    with pytest.raises(ValueError, match="win_left must"):
        tree(win_left=-1, positions=i)
    with pytest.raises(ValueError, match="positions must hold"):
        tree(win_left=3, positions=i[:3])
    with pytest.raises(ValueError, match="non-decreasing"):
        dsa.paged_tree_fwd(q, c, c, i.view(2, 2), m, actual_seq_lengths_query=[3, 1], actual_seq_lengths_kv=[4, 4])
    with pytest.raises(ValueError, match="for all S nodes"):
        dsa.paged_tree_fwd(torch.zeros(1, 65, 2, 64, dtype=torch.bfloat16), c, c, i.view(1, 4),
                           torch.zeros(1, 65, 1, dtype=torch.int64), actual_seq_lengths_kv=i[:1])
    accept = lambda x=torch.zeros(4, 8), tok=i, cu=i[:1], P=2: dsa.tree_accept(x, tok, i, actual_seq_lengths_query=cu,
                                                                             max_path=P)
    for kw, msg in [(dict(x=torch.zeros(4, 8, dtype=torch.float64)), "scores must be"), (dict(x=torch.zeros(4)), "scores must"),
                    (dict(x=i.view(2, 2)), "scores must"), (dict(tok=i[:3]), "tokens must"),
                    (dict(tok=torch.zeros(4)), "tokens must"), (dict(P=0), "max_path"), (dict(P=2**31), "max_path"),
                    (dict(P=2**70), "max_path"), (dict(cu=[3, 1]), "non-decreasing"), (dict(cu=i[:0]), "prefix sums")]:
        with pytest.raises(ValueError, match=msg):
            accept(**kw)
    with pytest.raises(ValueError, match="empty"):
        dsa.paged_commit([], i.view(1, 4), i[:1], i.view(1, 4), i[:1])


def test_meta_shapes(dsa):
    ops = dsa.load_torch_ops()
    m = dict(device="meta")
    ints = lambda *n: torch.empty(n, dtype=torch.int32, **m)
    p = ops.paged_plan(ints(3), ints(3), ints(3, 8), ints(9), ints(1), 16, 7, ints(7), 65)
    assert [tuple(x.shape) for x in p] == [(3,), (3,), (7,), (7,), (3,), (7, 2)] and p[5].dtype == torch.int64
    assert ops.paged_plan(ints(3), ints(3), ints(3, 8), ints(9), ints(1), 16, 7)[5].shape == (7, 0)
    ops.paged_free(ints(3), ints(3, 8), ints(9), ints(1), 16)
    q, c = torch.empty(7, 8, 64, dtype=torch.bfloat16, **m), torch.empty(4, 16, 2, 64, dtype=torch.bfloat16, **m)
    o, l = ops.paged_tree_fwd(q, c, c, ints(1, 4), p[5], ints(1), 0.1, ints(1))
    assert o.shape == q.shape and l.shape == (7, 8) and l.dtype == torch.float32
    a = ops.tree_accept(torch.empty(7, 100, **m), ints(7), ints(7), ints(2), 5)
    assert [tuple(x.shape) for x in a] == [(2,), (2, 5), (2, 5)] and a[1].dtype == torch.int32
    ops.paged_commit([c, c.clone()], ints(1, 4), ints(1), ints(1, 5), ints(1))


def test_lds_waits_cover_their_reads(tmp_path_factory):
    kernels, findings = asm_lds.check_asm(_asm(tmp_path_factory, "paged_tree.hip"))
    assert len(kernels) >= 8, kernels
    assert not findings, "\n".join(map(str, findings[:20]))


def test_oracle_of_the_plan():
    """By hand: three sequences, blocks of four, one page short."""
    table = [[5, -1, -1], [-1, -1, -1], [7, 8, -1]]
    count = [3]
    cu, kv, pos, slots, missing, mask = R.plan([3, 5, 1], [3, 0, 8], table, [1, 2, 3], count, 4, 11,
                                               parents=[-1, 0, 0] + [-1, 0, 1, 1, 7] + [-1] + [0, 0], max_nodes=4)
    assert table == [[5, 3, -1], [2, 1, -1], [7, 8, -1]] and count == [0]
    assert cu == [3, 8, 9] and kv == [6, 5, 9] and missing == [0, 0, 1]
    assert pos == [3, 4, 4, 0, 1, 2, 2, 0, 8, -1, -1]
    assert slots == [5 * 4 + 3, 3 * 4, 3 * 4 + 1, 8, 9, 10, 11, 4, -1, -1, -1]
    assert mask.view(-1).tolist() == [1, 3, 5, 1, 3, 7, 11, 16, 1, 0, 0]
    lists = [1, 2, 3]
    R.free([3, 0, 8], table, lists, count, 4)
    assert table == [[5, -1, -1], [-1, -1, -1], [7, 8, -1]] and lists == [1, 2, 3] and count == [3]


def test_oracle_of_acceptance():
    """0 -> 1 -> 4 by the choices; 2 has the right token but comes later; the last choice is new."""
    accepted, path, chosen = R.accept([9, 7, 3, 3, 2], [0, 9, 9, 7, 7], [-1, 0, 0, 0, 1], [5], 6)
    assert accepted.tolist() == [3] and path.tolist() == [[0, 1, 4, -1, -1, -1]] and chosen.tolist() == [[9, 7, 2, -1, -1, -1]]


def test_oracle_of_attention_on_a_chain():
    """A chain's masks are the causal rule of the dense attention."""
    import dense_layer_ref as dense

    g, rng = torch.Generator().manual_seed(1), random.Random(1)
    q, kc, vc = (torch.randn(s, generator=g).to(torch.bfloat16) for s in ((9, 4, 64), (8, 4, 2, 64), (8, 4, 2, 64)))
    table = torch.tensor([rng.sample(range(8), 4), rng.sample(range(8), 4)])
    mask = torch.cat([R.mask_words(R.ancestors([i - 1 for i in range(n)]), 1) for n in (5, 4)])
    args = ([0, 5], [5, 4], [5, 4], [11, 4], 0.125)
    for a, b in zip(R.attention(q, kc, vc, table, mask, *args), dense.attention(q, kc, vc, table, *args)):
        torch.testing.assert_close(a, b)
