"""A call that writes into a caller's tensor moves that tensor's version on, as torch's own in-place operations do: what autograd
saved of it is refused, and what was derived from it is known to be of older values."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Never:
    def __getattr__(self, name):
        return lambda *a: None


@pytest.fixture(params=["native", "checked"])
def path(request, monkeypatch):
    import h3mi
    if request.param == "checked":
        for m in (h3mi.fused, h3mi.gemm, h3mi.kvcache, h3mi.kvpages, h3mi.linear, h3mi.quant, h3mi.rope):
            monkeypatch.setattr(m, "_fast", _Never())
    return request.param


def _bf(*shape):
    return torch.randn(*shape, device=DEV).to(torch.bfloat16)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _calls(h):
    """(name, call, what it writes into, what it reads alone)"""
    S, N = 4, 128
    x, o, g, s1, sh, w, ridx = _bf(S, N), _bf(S, N), _bf(2, N), _bf(2, N), _bf(2, N), _bf(N), _i32(0, 1, 1, 0)
    norm = (w, 1e-6, ridx, s1, sh)
    hh = torch.empty_like(x)
    yield "gate_norm_mod_", lambda: h.gate_norm_mod_(x, o, g, *norm), [x], [o, g, w, ridx, s1, sh]
    yield "gate_norm_mod_q_", lambda: h.gate_norm_mod_q_(x, o, g, *norm), [x], [o, g, w]
    yield "gate_norm_mod_q_ with h", lambda: h.gate_norm_mod_q_(x, o, g, *norm, want_h=True), [x], [o, g, w]
    yield "gate_norm_mod_ex", lambda: h.gate_norm_mod_ex(x, o, g, *norm, h=hh), [x, hh], [o, g, w]
    yield "norm_mod_ex", lambda: h.norm_mod_ex(x, *norm, h=hh), [hh], [x, w]
    yield "norm_mod", lambda: h.norm_mod(x, *norm), [], [x, w]
    yield "gate_", lambda: h.gate_(x, o, g, ridx), [x], [o, g]
    q, k, tab = _bf(1, S, 2, 64), _bf(1, S, 2, 64), _bf(1, S, 32, 2, 2)
    yield "rms_rope_split_half_", lambda: h.rms_rope_split_half_(q, k, tab, w[:64], w[64:]), [q, k], [tab, w]
    rstd = torch.empty(2 * S * 2, device=DEV)
    yield "rms_rope_split_half_ with rstd_out", lambda: h.rms_rope_split_half_(q, k, tab, w[:64], w[64:], rstd_out=rstd), [q, k, rstd], [tab]
    positions, (freqs, _) = _i32(*range(S))[None], h.rotary_frequencies(64)
    yield "rotary_", lambda: h.rotary_(q, k, positions, freqs), [q, k], [positions, freqs]
    yield "rotary_ of q", lambda: h.rotary_(q, None, positions, freqs), [q], [k, positions, freqs]
    yield "rotary", lambda: h.rotary(q, k, positions, freqs), [], [q, k]
    tables, lens = _i32([1, 0]), _i32(S)
    for bits in (8, 4):
        cache = h.kv_cache(3, 2, 64, bits=bits)
        yield f"kv_write_ {bits}", lambda c=cache: h.kv_write_(c, q, k, tables, lens), list(cache), [q, k, tables, lens]
        yield f"kv_read {bits}", lambda c=cache: h.kv_read(c, tables, lens, 3), [], [*cache, tables, lens]
    pool, counts = h.kv_pool(5), _i32(3)
    yield "kv_extend_", lambda: h.kv_extend_(pool, tables, lens, 4, counts), [*pool, tables, lens], [counts]
    yield "kv_release_", lambda: h.kv_release_(pool, tables, lens, counts), [*pool, tables, lens], [counts]
    xq, xs = torch.empty(S, N, dtype=torch.int8, device=DEV), torch.empty(S, 1, device=DEV)
    yield "quantize_rowwise", lambda: h.quantize_rowwise(x, xq=xq, xs=xs), [xq, xs], [x]
    x256, q256 = _bf(S, 256), torch.empty(S, 256, dtype=torch.int8, device=DEV)
    yield "quantize_rowwise_convrot", lambda: h.quantize_rowwise_convrot(x256, xq=q256, xs=xs), [q256, xs], [x256]
    wq, ws, out, out32 = xq.clone().repeat(4, 1), torch.ones(16, 1, device=DEV), _bf(S, 16), torch.empty(S, 16, dtype=torch.int32, device=DEV)
    yield "int8_mm_scaled", lambda: h.int8_mm_scaled(xq, wq, xs, ws, out=out), [out], [xq, wq, xs, ws]
    yield "int8_mm_i32", lambda: h.int8_mm_i32(xq, wq, out=out32), [out32], [xq, wq]
    yield "w8a8_linear", lambda: h.w8a8_linear(x, wq, ws, out=out), [out], [x, wq, ws]


def test_what_is_written_moves_on(path):
    import h3mi
    for name, call, written, read in _calls(h3mi):
        before = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > v for t, v in zip(written, before[0])), name
        assert all(t._version == v for t, v in zip(read, before[1])), name


def test_autograd_sees_it(path):
    """x * a saves x for a's gradient: turning x in place before the backward pass is refused, not answered with x's new values."""
    import h3mi
    x, a = _bf(1, 3, 2, 64), _bf(64).requires_grad_()
    positions, (freqs, _) = _i32(5, 6, 7)[None], h3mi.rotary_frequencies(64)
    y = (x * a).sum()
    with torch.no_grad():
        h3mi.rotary_(x[:, :, :1], x[:, :, 1:], positions, freqs)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_no_stale_hand_off(path):
    """A quantization on offer is that of the tensor's values when it was offered."""
    import h3mi
    from h3mi import prequant
    x, ridx = _bf(4, 128), _i32(0, 0, 0, 0)
    o, g = _bf(4, 128), _bf(1, 128)
    q, qs = h3mi.quantize_rowwise(x)
    with prequant.offer(x, q, qs):
        assert prequant.take(x) is not None
        h3mi.gate_(x, o, g, ridx)
        assert prequant.take(x) is None


def test_inference_tensors(path):
    """Tensors of inference mode have no version: they are written to as before, in the mode and outside of it."""
    import h3mi
    with torch.inference_mode():
        calls = list(_calls(h3mi))
        for _, call, _, _ in calls:
            call()
    for _, call, _, _ in calls:
        call()
