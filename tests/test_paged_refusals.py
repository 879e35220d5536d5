"""What the paged-cache and prompt-attention entry points refuse, before anything is launched.  No GPU: validation never
dereferences a device pointer."""

import pytest
import torch

from nemotron_infer_b200 import _lib

BUF = 0x7F0000000000
OK, NULL, ALIGN, SHAPE, UNSUPPORTED = 0, 1, 2, 3, 5


def cache(**over):
    f = dict(k=BUF, v=BUF, k_page_stride=8 * 16 * 128, v_page_stride=8 * 16 * 128, num_pages=4, page_size=16, kv_heads=8, head_dim=128, dtype=0,
             k_scale=None, v_scale=None, scale_count=1, page_table=BUF, seq_lens=BUF, batch=2, max_pages=3)
    f.update(over)
    return _lib.PagedCache(**f)


BAD_CACHES = [
    (dict(page_size=12), UNSUPPORTED), (dict(page_size=4), UNSUPPORTED), (dict(page_size=2048), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED),
    (dict(dtype=2), UNSUPPORTED), (dict(num_pages=0), SHAPE), (dict(max_pages=0), SHAPE), (dict(kv_heads=0), SHAPE), (dict(batch=-1), SHAPE),
    (dict(k_page_stride=8 * 16 * 128 - 8), SHAPE), (dict(v_page_stride=8 * 16 * 128 + 4), ALIGN), (dict(k=BUF + 8), ALIGN), (dict(v=BUF + 2), ALIGN),
    (dict(page_table=BUF + 2), ALIGN), (dict(k_scale=BUF, scale_count=3, dtype=1), SHAPE), (dict(k_scale=BUF + 1, dtype=1), ALIGN), (dict(k_scale=BUF), UNSUPPORTED), (dict(v_scale=BUF), UNSUPPORTED), (dict(max_pages=1 << 28), UNSUPPORTED),
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(page_table=None), NULL), (dict(seq_lens=None), NULL),
]


def append(L, c, cu=BUF, tokens=5, k=BUF, kts=1024, khs=128, v=BUF, rope=None, rows=0, rot=0, q=None, q_heads=40, q_out=None, err=None):
    return L.nmt_kv_append_paged_bf16(c, cu, tokens, k, kts, khs, v, 1024, 128, rope, rows, rot, 0, q, 5120, 128, q_heads, q_out, 5120, 128, err, None)


def decode(L, c, q=BUF, hs=128, out=BUF, heads=40, scale=0.1, ws=BUF, err=None):
    return L.nmt_sdpa_decode_paged_bf16(c, q, 5120, hs, out, 5120, 128, heads, scale, err, ws, None)


@pytest.mark.parametrize("over,status", BAD_CACHES)
def test_bad_caches(built_lib, over, status):
    before = built_lib.nmt_launch_count()
    assert append(built_lib, cache(**over)) == status
    assert decode(built_lib, cache(**over)) == status
    assert built_lib.nmt_launch_count() == before


def test_append(built_lib):
    L = built_lib
    before = L.nmt_launch_count()
    assert append(L, None) == NULL
    assert append(L, cache(), tokens=0) == OK
    assert append(L, cache(batch=0), tokens=3) == OK
    assert append(L, cache(), tokens=-1) == SHAPE
    assert append(L, cache(), cu=None) == SHAPE                    # 5 tokens, 2 sequences, one each
    assert append(L, cache(), k=None) == NULL and append(L, cache(), v=None) == NULL
    assert append(L, cache(), k=BUF + 8) == ALIGN and append(L, cache(), kts=1020) == ALIGN and append(L, cache(), khs=132) == ALIGN
    assert append(L, cache(), kts=-1024) == UNSUPPORTED
    assert append(L, cache(), q=BUF, q_out=BUF) == NULL            # a query without a rotation
    assert append(L, cache(), q=BUF, rope=BUF, rows=10, rot=128) == NULL
    for rows, rot in ((0, 128), (10, 0), (10, 24), (10, 144)):
        assert append(L, cache(), rope=BUF, rows=rows, rot=rot) == SHAPE
    assert append(L, cache(), rope=BUF + 4, rows=10, rot=128) == ALIGN
    assert append(L, cache(), q=BUF, rope=BUF, rows=10, rot=128, q_out=BUF, q_heads=0) == SHAPE
    assert append(L, cache(), err=BUF + 2) == ALIGN
    assert L.nmt_launch_count() == before


def test_decode(built_lib):
    L = built_lib
    before = L.nmt_launch_count()
    assert decode(L, None) == NULL
    assert decode(L, cache(batch=0)) == OK
    assert decode(L, cache(), heads=12) == SHAPE and decode(L, cache(), heads=0) == SHAPE
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert decode(L, cache(), scale=scale) == SHAPE
    assert decode(L, cache(), q=None) == NULL and decode(L, cache(), out=None) == NULL and decode(L, cache(), ws=None) == NULL
    assert decode(L, cache(), q=BUF + 4) == ALIGN and decode(L, cache(), hs=60) == ALIGN and decode(L, cache(), ws=BUF + 8) == ALIGN
    assert L.nmt_sdpa_decode_paged_workspace_bytes(0, 40, 8, 128) == 0 and L.nmt_sdpa_decode_paged_workspace_bytes(1, 40, 7, 128) == 0
    assert L.nmt_sdpa_decode_paged_workspace_bytes(1, 40, 8, 128) > 0
    assert L.nmt_launch_count() == before


def test_operators_refuse_cpu_tensors(built_lib):
    from nemotron_infer_b200 import ops
    x = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    c = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16)
    t, n = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.kv_append_paged(x, x, c, c, t, n)
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.sdpa_decode_paged(x, c, c, t, n)


def test_descriptor_checks(built_lib):
    """The checks of shapes, types and layouts behind the tensor-level operators (they look at no data, so CPU tensors will do)."""
    from nemotron_infer_b200 import ops
    bf = torch.bfloat16
    c = torch.zeros(4, 8, 16, 128, dtype=bf)
    t, n = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    cpu = c.device
    ok = ops._paged_cache(c, c, t, n, None, None, cpu)
    assert (ok.num_pages, ok.kv_heads, ok.page_size, ok.head_dim, ok.batch, ok.max_pages, ok.dtype) == (4, 8, 16, 128, 2, 3, 0)
    both = torch.zeros(4, 2, 8, 16, 128, dtype=bf)
    assert ops._paged_cache(both[:, 0], both[:, 1], t, n, None, None, cpu).k_page_stride == 2 * 8 * 16 * 128
    one = torch.ones(1)
    for args in ((c.float(), c.float(), t, n, None, None), (c, c[:3], t, n, None, None), (c[0], c[0], t, n, None, None),
                 (c.transpose(1, 2), c.transpose(1, 2), t, n, None, None), (c, c, t.long(), n, None, None), (c, c, t[0], n, None, None),
                 (c, c, t, n[:1], None, None), (c, c, t, n.float(), None, None), (c, c, t.t(), n, None, None), (c, c, t, n, torch.ones(3), None),
                 (c, c, t, n, one.double(), None), (c, c, t, n, one, torch.ones(8)), (c, c.to(torch.float8_e4m3fn), t, n, None, None)):
        with pytest.raises(ValueError):
            ops._paged_cache(*args, cpu)
    with pytest.raises(ValueError, match="same device"):
        ops._paged_cache(c, c, t, n, None, None, torch.device("cuda", 0))
    x = torch.zeros(5, 8, 128, dtype=bf)
    assert ops._view3(x, "x", 5, 8, 128, x.device) == (1024, 128)
    assert ops._view3(torch.zeros(8, 5, 128, dtype=bf).transpose(0, 1), "x", 5, 8, 128, x.device) == (128, 640)
    for bad in (x.float(), x[0], x[:4], x[:, :7], x[..., :64], torch.zeros(5, 8, 256, dtype=bf)[..., ::2], x[..., None]):
        with pytest.raises(ValueError):
            ops._view3(bad, "x", 5, 8, 128, x.device)
    new, *strides = ops._result3(None, x.transpose(0, 1).contiguous().transpose(0, 1), "out", 5, 8, 128, x.device)
    assert new.is_contiguous() and strides == [1024, 128]
    for overlapping in (x[:1].expand(5, 8, 128), x[:, :1].expand(5, 8, 128), torch.zeros(4096, dtype=bf).as_strided((5, 8, 128), (8, 128, 1))):
        with pytest.raises(ValueError, match="overlap"):
            ops._result3(overlapping, x, "out", 5, 8, 128, x.device)


def test_rope_table_is_exact_at_far_positions():
    import math
    from nemotron_infer_b200 import ops
    t = ops.rope_table(200001, 64, device="cpu")
    assert t.shape == (200001, 64) and t.dtype == torch.float32
    for pos, i in ((200000, 0), (200000, 1), (131071, 5), (7, 31), (0, 3)):
        a = pos * 10000.0 ** (-2 * i / 64)
        assert abs(t[pos, i].item() - math.cos(a)) <= 2.0 ** -24 + 1e-9 and abs(t[pos, 32 + i].item() - math.sin(a)) <= 2.0 ** -24 + 1e-9


def prefill(L, q=BUF, qts=5120, k=BUF, kts=1024, v=BUF, out=BUF, cu=BUF, cu_k=None, batch=2, T=5, T_k=5, heads=40, kv=8, dim=128, scale=0.1, ws=None):
    return L.nmt_sdpa_prefill_bf16(q, qts, 128, k, kts, 128, v, 1024, 128, out, 5120, 128, cu, cu_k, batch, T, T_k, heads, kv, dim, scale, 1, ws, None)


def test_prefill(built_lib):
    L = built_lib
    before = L.nmt_launch_count()
    assert prefill(L, T=0) == OK and prefill(L, batch=0) == OK
    assert prefill(L, T=-1) == SHAPE and prefill(L, T_k=-1) == SHAPE and prefill(L, batch=-1) == SHAPE
    assert prefill(L, heads=12) == SHAPE and prefill(L, kv=0) == SHAPE
    assert prefill(L, dim=96) == UNSUPPORTED
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert prefill(L, scale=scale) == SHAPE
    assert prefill(L, cu=None) == SHAPE                            # one sequence, but batch 2
    assert prefill(L, cu=None, cu_k=BUF, batch=1) == SHAPE
    for name in ("q", "k", "v", "out"):
        assert prefill(L, **{name: None}) == NULL and prefill(L, **{name: BUF + 8}) == ALIGN
    assert prefill(L, qts=5124) == ALIGN and prefill(L, kts=-1024) == UNSUPPORTED
    assert prefill(L, cu=BUF + 2) == ALIGN and prefill(L, ws=BUF + 16) == ALIGN
    size = L.nmt_sdpa_prefill_workspace_bytes
    assert size(1, 16384, 16384, 40, 8, 128) == 0 and size(1, 200, 200, 40, 8, 128) == 0 and size(4, 100, 1000, 40, 7, 128) == 0
    assert size(4, 100, 20000, 40, 8, 128) > 0 and size(1, 1, 20000, 40, 8, 64) > 0
    assert prefill(L, T=1 << 31, T_k=1 << 31) == UNSUPPORTED
    assert L.nmt_launch_count() == before


def test_results_that_share_memory_with_inputs(built_lib):
    L = built_lib
    before = L.nmt_launch_count()
    for out in ("q", "k", "v"):
        at = {"q": BUF, "k": BUF + (1 << 20), "v": BUF + (2 << 20)}
        assert prefill(L, **at, out=at[out], kts=5120 if out == "k" else 1024, cu=None, batch=1, T=1, T_k=1) == UNSUPPORTED
    # keys behind the queries, as further heads, rotated in place: the key heads are read by others meanwhile
    rope = dict(rope=BUF + (1 << 24), rows=10, rot=128)
    assert append(L, cache(), k=BUF + 40 * 256, kts=40 * 128, q=BUF, q_heads=48, q_out=BUF, **rope) == UNSUPPORTED
    assert L.nmt_launch_count() == before
