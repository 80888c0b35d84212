"""CPU: what st_sample_logits, st_gemm_q4 and st_decode_sample refuse before any GPU call, the sizes they ask for, and the checks of
their Python callables."""
import ctypes as C

import pytest
import torch

from style_transfer_amd import _lib, ops


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def refused(L, rc, word, code=-1):
    text = L.st_last_error().decode()
    assert rc == code and word in text, (rc, text)


def settings(**kw):
    s = _lib.StSampleSettings(1.0, 0, 1.0, 0.0)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_sample_arguments(L):
    buf = C.create_string_buffer(4096)
    p = C.addressof(buf)
    call = lambda s=settings(), x=p, kind=0, ld=8, B=2, V=8, u=p, ids=p, ws=None, n=0: L.st_sample_logits(  # noqa: E731
        x, kind, ld, B, V, u, C.byref(s) if s is not None else None, ids, None, ws, n, None)
    refused(L, call(None), "settings")
    for kw, word in ((dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                     (dict(temperature=float("inf")), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=0.0), "top_p"),
                     (dict(top_p=1.5), "top_p"), (dict(top_p=float("nan")), "top_p"), (dict(min_p=-0.5), "min_p"), (dict(min_p=2.0), "min_p")):
        refused(L, call(settings(**kw)), word)
    refused(L, call(kind=3), "type")
    refused(L, call(B=-1), "B=")
    refused(L, call(V=0), "V=")
    refused(L, call(V=_lib.ST_SAMPLE_MAX_VOCAB + 1), "V=")
    refused(L, call(ld=-1), "ld=")
    refused(L, call(x=None), "NULL")
    refused(L, call(u=None), "NULL")
    refused(L, call(ids=None), "NULL")
    refused(L, call(x=p + 2), "size")
    refused(L, call(x=p + 1, kind=1), "size")
    refused(L, call(V=131072), "workspace too small", -3)
    refused(L, call(V=131072, ws=p, n=4096), "workspace too small", -3)
    refused(L, call(ws=p + 4, n=4096), "16 bytes")
    assert call(B=0, x=None, u=None, ids=None) == 0


def test_sample_workspace(L):
    assert L.st_sample_workspace_bytes(1, 9339) == 0 and L.st_sample_workspace_bytes(4096, 131072) == 0
    assert L.st_sample_workspace_bytes(1, 131072) > 0
    assert L.st_sample_workspace_bytes(0, 100) == 0 and L.st_sample_workspace_bytes(1, 1 << 20) == 0


def test_q4_arguments(L):
    buf = C.create_string_buffer(4096 + 16)
    p = (C.addressof(buf) + 15) // 16 * 16
    assert L.st_q4_packed_bytes(64, 128, 128, 0) == 4096 + 256 and L.st_q4_packed_bytes(64, 128, 128, 1) == 4096 + 512
    assert L.st_q4_packed_bytes(0, 128, 128, 0) == 0 and L.st_q4_packed_bytes(64, 128, 48, 0) == 0
    refused(L, L.st_pack_weight_q4(p, p, None, 4, 8, 16, p, None), "group")
    refused(L, L.st_pack_weight_q4(p, p, None, 0, 8, 32, p, None), "positive")
    refused(L, L.st_pack_weight_q4(p, None, None, 4, 8, 32, p, None), "NULL")
    refused(L, L.st_pack_weight_q4(p, p, None, 4, 8, 32, p + 4, None), "16 bytes")
    refused(L, L.st_quantize_weight_q4(p, 4, -8, 32, p, p, None, None), "positive")
    refused(L, L.st_quantize_weight_q4(None, 4, 8, 32, p, p, None, None), "NULL")
    w = _lib.StQ4Weight(p, 16, 8, 32, 0)
    call = lambda w=w, x=p, kind=0, ldx=8, M=2, y=p, ldy=16: L.st_gemm_q4(x, kind, ldx, M, C.byref(w) if w else None, None, y, ldy, None)  # noqa: E731
    refused(L, call(w=None), "weights")
    refused(L, call(w=_lib.StQ4Weight(p, 16, 8, 33, 0)), "group")
    refused(L, call(w=_lib.StQ4Weight(p, 16, 0, 32, 0)), "positive")
    refused(L, call(w=_lib.StQ4Weight(p + 8, 16, 8, 32, 0)), "16 bytes")
    refused(L, call(w=_lib.StQ4Weight(None, 16, 8, 32, 0)), "NULL")
    refused(L, call(kind=7), "type")
    refused(L, call(M=-1), "M=")
    refused(L, call(ldx=-8), "ldx")
    refused(L, call(ldy=15), "overlap")
    refused(L, call(x=None), "NULL")
    refused(L, call(y=p + 2), "size")
    assert call(M=0, x=None, y=None) == 0


def test_decode_sample_arguments(L):
    w = _lib.StDecoderWeights()
    w.d_model = 512
    s = settings()
    rc = L.st_decode_sample(C.byref(w), None, 0, 4, 60, 2, 3, 0, 0, 1, 0, C.byref(s), 0, None, 0, 0, None, None)
    refused(L, rc, "d_model")
    assert L.st_decode_sample_workspace_bytes(None, 4, 60, 0) == 0


def test_callables_refuse_cpu_tensors():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(ValueError):
        ops.sample_logits(x, u)
    with pytest.raises(ValueError):
        ops.quantize_weight_q4(x)
    with pytest.raises(ValueError):
        ops.pack_weight_q4(torch.zeros(2, 4, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.float16))


def test_values_in_common():
    """against the sets of addresses themselves"""
    def addresses(t):
        return {t.data_ptr() + 4 * (i * t.stride(0) + j) for i in range(t.shape[0]) for j in range(t.shape[1])}
    buf = torch.zeros(400)
    views = [buf.as_strided((m, n), (ld, 1), at) for m in (1, 3) for n, ld in ((5, 5), (5, 20), (12, 20), (7, 9)) for at in (0, 4, 5, 12, 26, 60)]
    for a in views:
        for b in views:
            common = bool(addresses(a) & addresses(b))
            got = ops._share_values(a, b)
            assert got or not common
    wide = torch.zeros(6, 20)
    assert not ops._share_values(wide[:, :8], wide[:, 8:]) and not ops._share_values(wide[:, 8:], wide[:, :8])
    assert ops._share_values(wide[:, :8], wide[:, 7:]) and ops._share_values(wide, wide) and not ops._share_values(wide[:0], wide)


def test_sample_decode_holds_as_many_rows_as_the_product_takes(L):
    """a small vocabulary and very many sentences: the logits held at a time are rows that st_gemm_q4 takes in one call"""
    up = lambda v: (v + 255) // 256 * 256  # noqa: E731
    for vocab, B, rows in ((60, 1100000, 65535 * 16 // 64 * 64), (60, 4096, 4096), (9339, 20000, 7232), (1, 1 << 21, 65535 * 16 // 64 * 64)):
        w = _lib.StDecoderWeights()
        w.d_model, w.n_heads, w.d_ff, w.n_layers, w.vocab, w.pe_rows = 256, 4, 1024, 2, vocab, 64
        more = L.st_decode_sample_workspace_bytes(C.byref(w), B, 2, 4) - L.st_decode_workspace_bytes_opt(C.byref(w), B, 2, 4)
        assert more == up(rows * vocab * 4) + 2 * up(B * 4)


def test_sample_rows_of_one_launch(L):
    """more rows than a launch has threads for are refused before it (2^32 threads, 256 to 1024 of them a row)"""
    buf = C.create_string_buffer(4096)
    p = C.addressof(buf)
    for V, most in ((1, (1 << 24) - 1), (2048, (1 << 24) - 1), (2049, (1 << 23) - 1), (32768, (1 << 23) - 1), (32769, (1 << 22) - 1), (524288, (1 << 22) - 1)):
        for B in (most + 1, (1 << 31) - 1):
            for kw in (dict(), dict(top_k=5), dict(temperature=0.0), dict(temperature_rows=p)):
                s = settings(**kw)
                refused(L, L.st_sample_logits(p, 1, 0, B, V, p, C.byref(s), p, None, None, 0, None), "at most %d rows" % most)


def test_values_in_common_of_two_types():
    """a row and a strided tensor of another type in one buffer, against the sets of bytes themselves"""
    def of(t):
        return {t.data_ptr() + t.element_size() * (i * t.stride(0) + j) + b for i in range(t.shape[0]) for j in range(t.shape[1]) for b in range(t.element_size())}
    buf = torch.zeros(200)
    half = buf.view(torch.bfloat16)
    rows = [buf.as_strided((1, n), (n, 1), at) for n in (3, 9) for at in (0, 4, 7, 20, 33)]
    for t in [half.as_strided((m, n), (ld, 1), at) for m in (1, 4) for n, ld in ((6, 6), (6, 20), (12, 44)) for at in (0, 7, 13)]:
        for r in rows:
            common = bool(of(t) & of(r))
            got = ops._share_values(t, r)
            assert got or not common
    wide = torch.zeros(6, 40).view(torch.bfloat16)
    assert not ops._share_values(wide[:, :40], wide.view(torch.float32)[2:3, 20:]) and ops._share_values(wide[:, :41], wide.view(torch.float32)[2:3, 20:])
