"""CPU checks of the dense layer's entries: argument checks of the C ABI (no kernel is launched), host tensors,
workspace sizes, registered schemas, the static check of the kernels' explicit LDS waits."""
import pytest
import torch

from test_lds_waits import _asm, asm_lds


def test_quant_matmul_c_checks(dsa):
    lib = dsa.load_library()
    call = lambda kind=1, M=4, N=8, K=64, x=16, ws=None: lib.dsa_quant_matmul(kind, x, 16, 16, 16, None, M, N, K, 16, ws, 0,
                                                                            None)
    for kw, msg in [(dict(kind=0), b"kind"), (dict(M=-1), b"M / N"), (dict(N=2**31), b"M / N"), (dict(K=0), b"K must"),
                    (dict(K=131072), b"K must"), (dict(x=None), b"null")]:
        assert call(**kw) == 1 and msg in lib.dsa_last_error_message()
    assert call(M=0) == 0 and call(N=0) == 0
    assert lib.dsa_quant_matmul_workspace_size(-1, 4, 64, 1) == 0
    assert lib.dsa_quant_matmul_workspace_size(4, 4, 0, 1) == 0


def test_norm_rope_c_checks(dsa):
    lib = dsa.load_library()

    def call(kind=1, q=16, qs=1024, wk=1, pos=16, T=4, H=4, G=2, D=64, R=64, eps=1e-6, slots=None, rows=0, v=None):
        return lib.dsa_qk_norm_rope(kind, q, qs, 16, 1024, v, 1024, None, None, wk, pos, 16, 16, 8, T, H, G, D, R, eps, 0,
                                    slots, rows, 16, 16, None, None)

    for kw, msg in [(dict(kind=3), b"kind"), (dict(wk=2), b"weights"), (dict(D=60), b"D must"), (dict(D=520), b"D must"),
                    (dict(R=24), b"R must"), (dict(R=80), b"R must"), (dict(T=-1), b"sizes"), (dict(eps=-1.0), b"eps"),
                    (dict(eps=float("nan")), b"eps"), (dict(pos=None), b"null"), (dict(q=24), b"16 bytes"),
                    (dict(qs=1020), b"strides"), (dict(slots=16, rows=8), b"null"), (dict(rows=2**31), b"sizes")]:
        assert call(**kw) == 1 and msg in lib.dsa_last_error_message(), kw
    assert call(T=0) == 0


def test_paged_gqa_c_checks(dsa):
    lib = dsa.load_library()

    def call(kind=1, q=16, T=4, B=2, S=2, H=8, G=2, D=64, nb=4, bs=16, mb=2, win=-1, scale=1.0, ws=16, nws=1 << 30, cu=None):
        return lib.dsa_paged_gqa_fwd(kind, q, 16, 16, 16, cu, None, 16, T, B, S, H, G, D, nb, bs, mb, 1, win, None, scale,
                                     16, 16, ws, nws, None)

    for kw, msg in [(dict(kind=0), b"kind"), (dict(D=96), b"D must"), (dict(H=7), b"multiple of kv_group"),
                    (dict(G=0), b"kv_group"), (dict(bs=0), b"page"), (dict(nb=2**31), b"page"),
                    (dict(mb=2**27), b"range"), (dict(T=5), b"B * S"), (dict(win=-2), b"win_left"),
                    (dict(scale=0.0), b"sm_scale"), (dict(scale=float("nan")), b"sm_scale"), (dict(q=None), b"null"),
                    (dict(q=18), b"16 bytes"), (dict(B=0, T=0), b"range"), (dict(T=2**30, S=2**29), b"range"),
                    (dict(nws=0), b"workspace"), (dict(ws=None), b"workspace")]:
        assert call(**kw) == 1 and msg in lib.dsa_last_error_message(), kw
    assert call(T=0, S=0) == 0
    assert lib.dsa_paged_gqa_workspace_size(1, 1, 64, 4, 128, 4160) > 0
    assert lib.dsa_paged_gqa_workspace_size(0, 1, 64, 4, 128, 4160) == 0
    assert lib.dsa_paged_gqa_workspace_size(1, 1, 64, 3, 128, 4160) == 0


def test_host_tensors_are_refused(dsa):
    i8, f = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    with pytest.raises(ValueError, match="HIP"):
        dsa.quant_matmul(i8, i8, f, f)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    t, pos = torch.zeros(8, 32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP"):
        dsa.qk_norm_rope(q, q, None, None, pos, t, t)
    c = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="HIP"):
        dsa.qk_norm_rope_paged(q, q, q, None, None, pos, t, t, c, c.clone(), pos)
    with pytest.raises(ValueError, match="HIP"):
        dsa.paged_gqa_fwd(q, c, c, pos.view(1, 4), actual_seq_lengths_query=pos[:1], actual_seq_lengths_kv=pos[:1])


def test_meta_shapes(dsa):
    ops = dsa.load_torch_ops()
    m = dict(device="meta")
    y = ops.quant_matmul(torch.empty(2, 5, 64, dtype=torch.int8, **m), torch.empty(24, 64, dtype=torch.int8, **m),
                         torch.empty(10, **m), torch.empty(24, **m), None, torch.float16)
    assert y.shape == (2, 5, 24) and y.dtype == torch.float16
    q, k = torch.empty(7, 8, 64, dtype=torch.bfloat16, **m), torch.empty(7, 2, 64, dtype=torch.bfloat16, **m)
    pos, tab = torch.empty(7, dtype=torch.int32, **m), torch.empty(9, 32, **m)
    qo, ko = ops.qk_norm_rope(q, k, None, None, pos, tab, tab)
    assert qo.shape == q.shape and ko.shape == k.shape
    c = torch.empty(4, 16, 2, 64, dtype=torch.bfloat16, **m)
    assert ops.qk_norm_rope_paged(q, k, k, None, None, pos, tab, tab, c, c.clone(), pos).shape == q.shape
    o, l = ops.paged_gqa_fwd(q, c, c, torch.empty(1, 4, dtype=torch.int32, **m), pos[:1], 0.1, pos[:1])
    assert o.shape == q.shape and l.shape == (7, 8) and l.dtype == torch.float32


@pytest.mark.parametrize("name,nkernels", [("paged_gqa.hip", 8), ("quant_matmul.hip", 6)])
def test_lds_waits_cover_their_reads(tmp_path_factory, name, nkernels):
    kernels, findings = asm_lds.check_asm(_asm(tmp_path_factory, name))
    assert len(kernels) >= nkernels, kernels
    assert not findings, "\n".join(map(str, findings[:20]))


def test_integers_past_32_bits_saturate(dsa):
    """A helper of the wrappers: what does not fit 32 bits stays at its end of them."""
    cast = dsa._lib.saturated_int32
    top, low = 2**31 - 1, -2**31
    for dtype, given, want in [(torch.int64, [2**32 + 5, -2**63, 2**63 - 1, -7, 2**31, 4], [top, low, top, -7, top, 4]),
                               (torch.uint32, [2**32 - 1, 2**31, 9], [top, top, 9]),
                               (torch.uint64, [2**64 - 1, 2**63 + 5, 2**32, 9], [top, top, top, 9]),
                               (torch.int32, [low, top], [low, top]), (torch.uint16, [65535], [65535]),
                               (torch.uint8, [255], [255]), (torch.int8, [-1], [-1])]:
        got = cast(torch.tensor(given, dtype=dtype))
        assert got.dtype == torch.int32 and got.tolist() == want, dtype


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.bool, torch.complex64])
def test_block_tables_hold_integers(dsa, dtype):
    q, c = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    n = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="block_table must hold integers"):
        dsa.paged_gqa_fwd(q, c, c, torch.zeros(1, 4, dtype=dtype), actual_seq_lengths_query=n, actual_seq_lengths_kv=n)


@pytest.mark.parametrize("sums", [[3, 1], torch.tensor([3, 0]), torch.tensor([2**32, 4]),
                                  torch.tensor([3, -1], dtype=torch.int32)])
def test_prefix_sums_on_the_host_do_not_decrease(dsa, sums):
    q, c = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    call = lambda cu: dsa.paged_gqa_fwd(q, c, c, torch.zeros(2, 4, dtype=torch.int32), actual_seq_lengths_query=cu,
                                        actual_seq_lengths_kv=[4, 4])
    with pytest.raises(ValueError, match="non-decreasing"):
        call(sums)
    with pytest.raises(ValueError, match="HIP"):  # the next check: host tensors
        call([3, 3])


def test_norms_need_caches_only_for_rows(dsa):
    """Null caches are refused where they have rows."""
    lib = dsa.load_library()
    call = lambda rows: lib.dsa_qk_norm_rope(1, 16, 128, 16, 128, 16, 128, None, None, 1, 16, 16, 16, 8, 4, 1, 1, 64, 64,
                                             1e-6, 0, 16, rows, 16, None, None, None)
    assert call(8) == 1 and b"null" in lib.dsa_last_error_message()


def test_grids_past_32_bits_of_threads_are_refused(dsa):
    """Sizes within every other bound whose launch would pass 2^32 threads."""
    lib = dsa.load_library()
    refused = lambda rc: rc == 1 and b"range" in lib.dsa_last_error_message()
    qmm = lambda M, N, K, x=16, ws=None, n=0: lib.dsa_quant_matmul(1, x, 16, 16, 16, None, M, N, K, 16, ws, n, None)
    assert refused(qmm(1, 2**27 + 16, 16))  # 16 channels a workgroup of 512
    assert refused(qmm(2**26, 32, 17, ws=16, n=2**62))  # copies, a wave a row
    assert refused(qmm(2**26, 32, 16, x=24, ws=16, n=2**62))
    rope = lambda T, H, D: lib.dsa_qk_norm_rope(1, 16, H * D, 16, H * D, None, 0, None, None, 1, 16, 16, 16, 8, T, H, 0, D, 0,
                                                1e-6, 0, None, 0, 16, 16, None, None)
    assert refused(rope(2**24, 127, 512))
    # Decode tiles of 256 threads: a slot for each of 65535 sequences and their rows, in each of 1024 groups.
    attn = lambda T, B, H, G: lib.dsa_paged_gqa_fwd(1, 16, 16, 16, 16, 16, None, 16, T, B, 0, H, G, 64, 4, 16, 2, 1, -1, None,
                                                    1.0, 16, 16, 16, 2**62, None)
    assert refused(attn(2**15, 65535, 4096, 4096))
    assert lib.dsa_paged_gqa_workspace_size(2**15, 65535, 4096, 4096, 64, 32) == 0
