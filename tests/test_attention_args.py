"""Argument rules of the attention and KV-page launchers (include/b200_layer_ops.h, part 5), without a device: what the
contract forbids is cudaErrorInvalidValue, a call it allows is cudaErrorInvalidDeviceFunction before gpu_ops_init, and
nothing is launched either way."""
import ctypes as C

import pytest

from rocm_hip_b200 import _lib

BAD, NODEV = _lib.cudaErrorInvalidValue, _lib.cudaErrorInvalidDeviceFunction
Q, K, V, O, S, P, L, W = (C.c_void_p(0x10000 * (i + 1)) for i in range(8))   # never read: no call gets that far


@pytest.fixture(scope="module")
def lib():
    import torch
    lib = _lib.load()
    if torch.cuda.is_available():
        lib.gpu_ops_free()
    n = lib.b200_launch_count()
    yield lib
    assert lib.b200_launch_count() == n
    if torch.cuda.is_available():
        assert lib.gpu_ops_init(b"gpu_ops.co") == 0


PROMPT = dict(q=Q, k=K, v=V, out=O, seq_start=S, n_seqs=3, T=100, n_q=8, n_kv=2, head_dim=128, q_stride=0, k_stride=0, v_stride=0,
              scale=0.1, stream=None)


@pytest.mark.parametrize("name", ["gpu_attn_prompt_bf16", "gpu_attn_prompt_f16"])
def test_prompt(lib, name):
    call = lambda **kw: getattr(lib, name)(*{**PROMPT, **kw}.values())  # noqa: E731
    for ok in (dict(), dict(seq_start=None, n_seqs=1), dict(head_dim=64), dict(head_dim=256), dict(n_q=2), dict(n_kv=8),
               dict(q_stride=1536, k_stride=1536, v_stride=1536), dict(T=1), dict(n_seqs=1000), dict(n_q=10)):
        assert call(**ok) == NODEV, ok
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(seq_start=None), dict(n_seqs=0), dict(T=0), dict(T=-1),
                dict(T=(1 << 27) + 1), dict(n_seqs=2**31 - 1), dict(n_q=7), dict(n_q=0), dict(n_kv=0), dict(n_kv=-2), dict(head_dim=96), dict(head_dim=512),
                dict(head_dim=0), dict(q_stride=1000), dict(q_stride=1020), dict(k_stride=255), dict(v_stride=-256), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=Q), dict(out=V),
                dict(q=C.c_void_p(0x10008)), dict(out=C.c_void_p(0x40002))):
        assert call(**bad) == BAD, bad


DECODE = dict(q=Q, K=K, V=V, kv_stride=256, kv_shift=4, kv_bstride=8192, n_pages=50, pages=P, max_pages=20, lens=L, prefix_len=0,
              out=O, n_q=8, n_kv=2, head_dim=128, B=5, scale=0.1, scratch=W, scratch_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("name", ["gpu_attn_decode", "gpu_attn_decode_bf16"])
def test_decode(lib, name):
    call = lambda **kw: getattr(lib, name)(*{**DECODE, **kw}.values())  # noqa: E731
    for ok in (dict(), dict(prefix_len=16), dict(prefix_len=320), dict(kv_shift=0), dict(kv_shift=30, max_pages=1), dict(kv_stride=264),
               dict(B=1), dict(n_q=2), dict(n_q=64)):
        assert call(**ok) == NODEV, ok
    need = lib.gpu_attn_decode_scratch_bytes(8, 2, 128, 5, 0)
    assert need > 0 and call(scratch_bytes=need) == NODEV
    for bad in (dict(q=None), dict(K=None), dict(V=None), dict(pages=None), dict(lens=None), dict(out=None), dict(scratch=None),
                dict(scratch_bytes=need - 1), dict(scratch=C.c_void_p(0x80004)), dict(prefix_len=-16), dict(prefix_len=8),
                dict(prefix_len=336), dict(kv_shift=-1), dict(kv_shift=31), dict(kv_stride=248), dict(kv_stride=260),
                dict(kv_bstride=8190), dict(kv_bstride=-8), dict(n_pages=0), dict(max_pages=0), dict(B=0), dict(n_q=9), dict(n_kv=0),
                dict(head_dim=80), dict(scale=0.0), dict(scale=float("inf")), dict(out=Q), dict(K=C.c_void_p(0x20008))):
        assert call(**bad) == BAD, bad
    for bad in ((7, 2, 128, 5, 0), (8, 0, 128, 5, 0), (8, 2, 100, 5, 0), (8, 2, 128, 0, 0), (8, 2, 128, 5, -1)):
        assert lib.gpu_attn_decode_scratch_bytes(*bad) == 0, bad


PAGES = dict(table=Q.value, lens=K.value, refs=V.value, info=O.value, work=W.value, n_seqs=4, max_pages=8, n_pages=30, page_shift=4,
             pool=P.value, page_bytes=4096, n_parts=1, part_stride=0)


def test_pages(lib):
    s = lambda **kw: _lib.b200_kv_pages(*{**PAGES, **kw}.values())  # noqa: E731
    calls = [lambda kv: lib.gpu_kv_pages_fork(C.byref(kv), L, None), lambda kv: lib.gpu_kv_pages_resize(C.byref(kv), L, S, 10, None),
             lambda kv: lib.gpu_kv_pages_compact(C.byref(kv), None)]
    for call in calls:
        for ok in (dict(), dict(n_parts=3, part_stride=30 * 4096), dict(page_shift=0), dict(page_bytes=16)):
            assert call(s(**ok)) == NODEV, ok
        for bad in (dict(table=None), dict(lens=None), dict(refs=None), dict(info=None), dict(work=None), dict(pool=None),
                    dict(pool=0x10004), dict(n_seqs=0), dict(max_pages=0), dict(n_pages=0), dict(page_shift=-1),
                    dict(page_shift=27), dict(n_seqs=1 << 20, max_pages=1 << 12), dict(page_bytes=0), dict(page_bytes=24), dict(n_parts=0), dict(n_parts=2, part_stride=4096),
                    dict(n_parts=2, part_stride=30 * 4096 + 8)):
            assert call(s(**bad)) == BAD, bad
    assert lib.gpu_kv_pages_fork(None, L, None) == BAD
    assert lib.gpu_kv_pages_fork(C.byref(s()), None, None) == BAD
    assert lib.gpu_kv_pages_fork(C.byref(s()), K, None) == BAD
    assert lib.gpu_kv_pages_resize(C.byref(s()), K, S, 10, None) == BAD
    assert lib.gpu_kv_pages_resize(C.byref(s()), None, S, 10, None) == BAD
    assert lib.gpu_kv_pages_resize(C.byref(s()), L, S, -1, None) == BAD
    assert lib.gpu_kv_pages_resize(C.byref(s()), L, None, 0, None) == NODEV
    assert lib.gpu_kv_pages_work_ints(0, 5) == 0 and lib.gpu_kv_pages_work_ints(5, 0) == 0
    assert lib.gpu_kv_pages_work_ints(4, 30) >= 3 * 30


def test_struct_layout(tmp_path):
    """The ctypes mirror has the C compiler's offsets."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [f[0] for f in _lib.b200_kv_pages._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include "b200_layer_ops.h"\n#include <stdio.h>\nint main(void){printf("%zu", sizeof(b200_kv_pages));\n'
                   + "".join('printf(" %%zu", offsetof(b200_kv_pages, %s));\n' % f for f in fields) + "return 0;}\n")
    exe = tmp_path / "o"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), "-I/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(_lib.b200_kv_pages)] + [getattr(_lib.b200_kv_pages, f).offset for f in fields]


@pytest.mark.parametrize("n_q,n_kv,D", [(16, 4, 256), (16, 8, 128), (40, 8, 128), (8, 1, 64), (5, 1, 128), (128, 16, 256), (64, 2, 64)])
def test_scratch_of_the_largest_call_serves_the_smaller_ones(lib, n_q, n_kv, D):
    """One workspace for the largest batch behind the longest prefix: every call with fewer sequences or a shorter prefix takes it."""
    Bs = sorted({*range(1, 40), *range(120, 135), 200, 255, 256, 257, 300, 511, 512, 1000})
    prefixes = sorted({0, 16, 240, 256, 272, 1024, 2432, 8192, 8208, 16384, 32768, 131072, *range(256, 5000, 208)})
    need = [[lib.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, B, p) for p in prefixes] for B in Bs]
    for i, row in enumerate(need):
        for j, n in enumerate(row):
            assert n > 0 and (i == 0 or need[i - 1][j] <= n) and (j == 0 or row[j - 1] <= n), (Bs[i], prefixes[j])
    kw = dict(DECODE, n_q=n_q, n_kv=n_kv, head_dim=D, kv_stride=n_kv * D, kv_bstride=32 * n_kv * D, max_pages=1 << 20)
    for B, p in ((257, 8192), (129, 2432), (1000, 131072)):
        most = lib.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, B, p)
        for b in Bs:
            for q in prefixes:
                if b <= B and q <= p:
                    for name in ("gpu_attn_decode", "gpu_attn_decode_bf16"):
                        assert getattr(lib, name)(*dict(kw, B=b, prefix_len=q, scratch_bytes=most).values()) == NODEV, (B, p, b, q)
    assert lib.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, 8, 2**31 - 1) >= lib.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, 8, 2**31 - 6000)


def test_prefixes_beyond_what_a_sequence_can_hold(lib):
    """Prefixes up to the largest int: allowed where the page lists can hold them, and never more than an int on the way."""
    call = lambda **kw: lib.gpu_attn_decode(*{**DECODE, **kw}.values())  # noqa: E731
    for shift, prefix in ((0, 2**31 - 1), (0, 2**31 - 128), (0, 2**31 - 4097), (0, 2**31 - 4095), (7, 2**31 - 128), (30, 2**30)):
        assert call(kv_shift=shift, prefix_len=prefix, max_pages=2**31 - 1 >> shift) == NODEV, (shift, prefix)
