"""What the Python mirror of the attention and KV-page calls refuses before anything is launched: index arrays of another type,
too short, in strides or on another device, and rows with less memory behind them than the call reads or writes."""
import pytest
import torch

from rocm_hip_b200 import ops as mirror

BF, F16, I32 = torch.bfloat16, torch.float16, torch.int32


def test_index_arrays():
    ok = torch.zeros(6, dtype=I32)
    mirror._ints("x", ok, 6, -1)
    mirror._ints("x", ok.view(2, 3), 5, -1)
    mirror._ints("x", ok[2:], 4, -1)
    mirror._ints("x", ok[:0], 0, -1)
    for t, n, error in ((ok.long(), 6, TypeError), (ok.float(), 6, TypeError), (ok.to(torch.int16), 6, TypeError), (ok, 7, ValueError),
                        (ok[::2], 3, ValueError), (ok.view(2, 3).t(), 6, ValueError), (ok[3:], 4, ValueError)):
        with pytest.raises(error, match="x"):
            mirror._ints("x", t, n, -1)
    with pytest.raises(ValueError):
        mirror._ints("x", ok, 6, 0)


def test_rows():
    buf = torch.zeros(5, 8)
    room = lambda t, values, contiguous=False: mirror._room("x", t, 4 * values, -1, contiguous)  # noqa: E731
    assert room(buf, 40, True) == buf.data_ptr()
    assert room(buf[:, 2:4], 4 * 8 + 2) == buf.data_ptr() + 8     # a column block: to its last row's end
    room(buf[:, 2:4], 38)                                         # (what lies behind it is the buffer's too)
    room(buf[1], 32)                                              # a view's first value, and all behind it
    for bad in ((buf, 41), (buf[:, 2:4], 39), (buf[1], 33), (buf[:, 2:4], 1, True), (buf[4:], 9, True)):
        with pytest.raises(ValueError, match="x"):
            room(*bad)
    with pytest.raises(ValueError):
        mirror._room("x", buf, 1, 0)


@pytest.mark.gpu
def test_prompt_tensors(ops):
    T, D = 40, 128
    q, k, v = (torch.randn(T, n * D, device="cuda").to(BF) for n in (2, 1, 1))
    ss = torch.tensor([0, 30, T], dtype=I32, device="cuda")

    def call(q=q, k=k, v=v, out=None, ss=ss, n=2, **kw):
        out = torch.empty(T, 2 * D, dtype=BF, device="cuda") if out is None else out
        ops.gpu_attn_prompt(q, k, v, out, ss, n, T, 2, 1, D, 0.1, **kw)
        return out

    want = call()
    wide = torch.zeros(T, 4 * D + 8, dtype=BF, device="cuda")
    wide[:, :2 * D], wide[:, 2 * D:3 * D], wide[:, 3 * D:4 * D] = q, k, v
    st = wide.stride(0)
    fused = dict(q=wide[:, :2 * D], k=wide[:, 2 * D:3 * D], v=wide[:, 3 * D:4 * D], q_stride=st, k_stride=st, v_stride=st)
    assert torch.equal(call(**fused), want)
    before = ops.launch_count()
    for bad in (dict(ss=ss.long()), dict(ss=ss.float())):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(ss=ss[:2]), dict(ss=ss.cpu()), dict(ss=torch.zeros(6, dtype=I32, device="cuda")[::2]), dict(k=k.cpu()),
                dict(out=want.cpu()), dict(q=q[1:]), dict(k=k[:39]), dict(v=v[1:]), dict(out=torch.empty(T - 1, 2 * D, dtype=BF, device="cuda")),
                dict(q=wide[:, :2 * D]), dict(out=wide[:, :2 * D]), dict(fused, q=wide[1:, :2 * D]), dict(fused, v_stride=st + 8)):
        with pytest.raises(ValueError):
            call(**bad)
    assert ops.launch_count() == before


@pytest.mark.gpu
def test_decode_tensors(ops):
    B, n_q, n_kv, D, page, n_pages, max_pages = 3, 4, 2, 64, 16, 10, 4
    kv = n_kv * D
    pool = torch.randn(n_pages, 2, page, kv, device="cuda").to(F16)
    q = torch.randn(B, n_q * D, device="cuda")
    table = torch.arange(B * max_pages, dtype=I32, device="cuda").view(B, max_pages) % n_pages
    lens = torch.tensor([20, 64, 3], dtype=I32, device="cuda")
    scratch = torch.empty(ops.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, B), dtype=torch.uint8, device="cuda")

    def call(q=q, K=pool, V=None, pages=table, lens=lens, out=None, scratch=scratch, n=n_pages):
        out = torch.empty_like(q) if out is None else out
        ops.gpu_attn_decode(q, K, pool[:, 1] if V is None else V, kv, 4, 2 * page * kv, n, pages, max_pages, lens, 0, out, n_q, n_kv, D, B,
                            0.1, scratch)
        return out

    want = call()
    assert torch.equal(call(scratch=None), want) and torch.equal(call(V=pool[0, 1]), want)
    before = ops.launch_count()
    for bad in (dict(pages=table.long()), dict(lens=lens.long()), dict(lens=lens.float()), dict(K=pool.float()), dict(q=q.half())):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(pages=table[:2]), dict(pages=table.t()), dict(pages=table.cpu()), dict(lens=lens[:2]), dict(lens=lens.cpu()), dict(K=pool.cpu()),
                dict(V=pool.cpu()), dict(K=pool[1:]), dict(V=pool[:9, 1].clone()), dict(n=n_pages + 1), dict(scratch=scratch.cpu()),
                dict(q=q[:2], out=torch.empty_like(q)), dict(out=torch.empty(2, n_q * D, device="cuda")), dict(out=want.cpu()),
                dict(out=torch.empty(B, 2 * n_q * D, device="cuda")[:, :n_q * D])):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ops.LayerOpError):
        call(scratch=scratch[:-1])
    assert ops.launch_count() == before


@pytest.mark.gpu
def test_page_tensors(ops):
    n_seqs, max_pages, n_pages = 4, 6, 20
    z = lambda *n: torch.zeros(*n, dtype=I32, device="cuda")  # noqa: E731
    arrays = dict(table=z(n_seqs, max_pages) - 1, lens=z(n_seqs), refs=z(n_pages), info=z(4), page_shift=2,
                  pool=torch.zeros(n_pages, 16, device="cuda"), page_bytes=64)
    kv = ops.KvPages(**arrays)
    for bad in (dict(lens=arrays["lens"].long()), dict(table=arrays["table"].long()), dict(info=arrays["info"].float())):
        with pytest.raises(TypeError):
            ops.KvPages(**{**arrays, **bad})
    for bad in (dict(lens=z(3)), dict(info=z(3)), dict(refs=z(n_pages).cpu()), dict(table=arrays["table"].cpu()), dict(table=arrays["table"].t()),
                dict(refs=z(n_pages + 1)), dict(page_bytes=80), dict(pool=arrays["pool"].cpu()), dict(pool=arrays["pool"][1:])):
        with pytest.raises(ValueError):
            ops.KvPages(**{**arrays, **bad})
    ops.gpu_kv_pages_resize(kv, torch.tensor([5, 0, 0, 0], dtype=I32, device="cuda"), z(5))
    want = [t.clone() for t in (kv.table, kv.lens, kv.refs, kv.info)]
    before = ops.launch_count()
    ids = torch.tensor([7, 0, 0, 0], dtype=I32, device="cuda")
    parents = torch.tensor([-1, 0, -1, -1], dtype=I32, device="cuda")
    for call in (lambda: ops.gpu_kv_pages_resize(kv, ids.long()), lambda: ops.gpu_kv_pages_resize(kv, ids, z(9).long()),
                 lambda: ops.gpu_kv_pages_fork(kv, parents.long())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ops.gpu_kv_pages_resize(kv, ids[:3]), lambda: ops.gpu_kv_pages_resize(kv, ids.cpu()),
                 lambda: ops.gpu_kv_pages_resize(kv, ids, z(9).cpu()), lambda: ops.gpu_kv_pages_resize(kv, ids, z(9)[::2]),
                 lambda: ops.gpu_kv_pages_fork(kv, parents[:3]), lambda: ops.gpu_kv_pages_fork(kv, parents.cpu())):
        with pytest.raises(ValueError):
            call()
    assert ops.launch_count() == before
    assert all(torch.equal(a, b) for a, b in zip(want, (kv.table, kv.lens, kv.refs, kv.info)))
