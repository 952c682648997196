"""CPU checks of the C ABI boundary: the library loads and exports every entry point that
include/*.h declares, and argument validation rejects bad calls without touching a GPU."""
import ctypes
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def _declared():
    names = set()
    for h in (ROOT / "include").glob("*.h"):
        text = h.read_text()
        text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
        names.update(re.findall(r"\b(spar_(?:cuda|b200)_\w+)\s*\(", text))
    return sorted(names)


def test_headers_declare_entry_points():
    names = _declared()
    assert "spar_cuda_launch_adamw" in names and "spar_b200_gemm" in names
    assert len([n for n in names if n.startswith("spar_cuda_")]) == 23


def test_library_exports_every_declared_symbol():
    from spar_b200 import _lib

    lib = _lib.load()
    missing = [n for n in _declared() if not hasattr(lib, n)]
    assert not missing, f"not exported: {missing}"


def test_binding_table_matches_headers():
    from spar_b200 import _lib

    bound = set(_lib.exported_symbols())
    missing = [n for n in _declared() if n not in bound]
    assert not missing, f"no ctypes signature for: {missing}"


def test_invalid_arguments_rejected_without_gpu():
    """Argument validation runs before any CUDA call (reference convention: code 1)."""
    from spar_b200 import _lib, ops

    lib = _lib.load()
    st = lib.spar_b200_layernorm_forward(None, None, None, None, None, None, 4, 6, 1e-5, 0, None)
    assert st.code == 1  # cols not a multiple of 4
    st = lib.spar_b200_gemm(ctypes.byref(ops.gemm_desc(0, 0, 0, None, 0, None, 0, None, 0)), 0, None)
    assert st.code == 1
    st = lib.spar_b200_adamw_clipped(None, 0, None, 1.0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, 0,
                                     None)
    assert st.code == 1
    st = lib.spar_b200_cross_entropy_forward_backward(None, None, None, None, 8, 4, 4, 1, 1.0, None,
                                                      0, None)
    assert st.code == 1


def test_layernorm_backward_rejects_misaligned_pointers_without_gpu():
    """The LayerNorm backward reads x, dy, gamma and writes dx as float4: a base pointer that is
    not 16-byte aligned is an invalid argument (code 1), checked before any CUDA call."""
    from spar_b200 import _lib

    lib = _lib.load()
    good, bad = 1 << 20, (1 << 20) + 4  # never dereferenced: validation fails first
    for fn in (lib.spar_b200_layernorm_backward, lib.spar_b200_layernorm_backward_noalloc):
        for k in range(4):  # dx, dy, x, gamma in turn
            ptrs = [good] * 4
            ptrs[k] = bad
            dx, dy, x, g = ptrs
            st = fn(dx, good, good, dy, x, g, good, good, 8, 64, 0, 0, 0, None)
            assert st.code == 1, (fn, k)


def test_zero_count_calls_succeed():
    """Zero-count calls return success without launching (reference cuda_kernels.cu convention)."""
    from spar_b200 import _lib

    lib = _lib.load()
    assert lib.spar_b200_gelu_forward(None, None, 0, 0, None).code == 0
    assert lib.spar_b200_layernorm_forward(None, None, None, None, None, None, 0, 8, 1e-5, 0,
                                           None).code == 0
    assert lib.spar_b200_causal_softmax_forward(None, None, 0, 16, 16, 1.0, 0, 0, None).code == 0


def test_error_string_and_version():
    from spar_b200 import _lib

    lib = _lib.load()
    if hasattr(lib, "spar_cuda_error_string"):
        assert lib.spar_cuda_error_string(0)
    if hasattr(lib, "spar_b200_version"):
        assert b"spar_b200" in lib.spar_b200_version()


def test_product_does_not_import_oracle():
    """The product package must never route through the CPU oracle."""
    for p in (ROOT / "spar_b200").rglob("*.py"):
        src = p.read_text()
        assert not re.search(r"^\s*(from|import)\s+oracle", src, re.M), p


if __name__ == "__main__":
    pytest.main([__file__])


def test_warmup_cosine_entry_point_matches_reference_fixture():
    """spar_b200_warmup_cosine reproduces the reference schedule bit for bit."""
    import numpy as np

    from spar_b200.lm import warmup_cosine

    f = np.load(ROOT / "tests" / "golden" / "schedule.npz")
    for s, lr in zip(f["steps"], f["lr"]):
        assert warmup_cosine(3e-4, 3e-5, 100, 900, int(s)) == lr


def test_rotary_and_window_attention_refuse_bad_calls_without_gpu():
    """Sizes, strides, tags and pointers are checked before any CUDA call (code 1); zero-count calls
    succeed."""
    from spar_b200 import _lib

    lib = _lib.load()
    at = 1 << 20  # never dereferenced: validation fails first

    def rotary(**k):
        strides = {f"{n}_{part}": x for n in ("q", "k", "q_out", "k_out", "dq", "dk")
                   for part, x in (("batch", 1024), ("token", 256), ("head", 64))}
        base = dict(strides, dtype=0, layout=1, batch=2, seq=3, heads=4, kv_heads=2, head_dim=64, rotary_dim=32,
                    table=at, table_rows=3, q=at, k=at + 4096, q_out=at, k_out=at + 4096, q_weight=at,
                    k_weight=at, epsilon=1e-6, dq=at + 8192, dk=at + 12288, dq_weight=at,
                    dk_weight=at + 256, scratch=at)
        return ctypes.byref(_lib.SparB200Rotary(**{**base, **k}))

    for bad in (dict(dtype=2), dict(layout=2), dict(head_dim=0), dict(head_dim=257), dict(rotary_dim=31),
                dict(rotary_dim=66), dict(rotary_dim=0), dict(heads=0), dict(table=None), dict(q=None),
                dict(k_out=None), dict(table_rows=2), dict(start=1), dict(start=2 ** 64 - 1), dict(q=at + 2),
                dict(batch=1 << 20, seq=1 << 20), dict(batch=1 << 40, seq=1 << 40),
                dict(q_out_token=0), dict(k_out_head=0),  # rows of an output on one another
                dict(q_out=at + 4096), dict(k_out=at), dict(q_out_token=512), dict(k_out_batch=2048),
                dict(q_out=at + 16384, k_out=at + 16384),  # not element by element in place
                dict(positions=at + 2), dict(invalid=at + 1)):
        assert lib.spar_b200_rotary(rotary(**bad), 0, None).code == 1, bad
        assert lib.spar_b200_qk_norm_rotary_forward(rotary(**bad), 0, None).code == 1, bad
        assert lib.spar_b200_qk_norm_rotary_backward(rotary(**bad), 0, None).code == 1, bad
    for bad in (dict(q_weight=None), dict(k_weight=at + 2), dict(epsilon=-1.0), dict(epsilon=float("nan"))):
        assert lib.spar_b200_qk_norm_rotary_forward(rotary(**bad), 0, None).code == 1, bad
    for bad in (dict(dq_weight=None), dict(dk_weight=None), dict(scratch=None), dict(scratch=at + 4),
                dict(dk=None), dict(dk_weight=at), dict(dk_weight=at + 252), dict(dq_weight=at + 2),
                dict(q_out=at + 12288), dict(q_out=at + 8192, dq_head=128)):
        assert lib.spar_b200_qk_norm_rotary_backward(rotary(**bad), 0, None).code == 1, bad
    assert lib.spar_b200_rotary(None, 0, None).code == 1
    assert lib.spar_b200_rotary(rotary(seq=0, table=None, q=None, q_out=None), 0, None).code == 0
    for args in ((at, 4, 31, 1e4, 0), (at, 4, 0, 1e4, 0), (at, 4, 32, 0.0, 0), (None, 4, 32, 1e4, 0),
                 (at + 4, 4, 32, 1e4, 0), (at, 4, 258, 1e4, 0), (at, 4, 32, float("inf"), 0)):
        assert lib.spar_b200_rotary_table(*args, None, 0, None).code == 1, args
    assert lib.spar_b200_rotary_table(None, 0, 32, 1e4, 0, None, 0, None).code == 0

    def window(**k):
        strides = {f"{n}_{part}": x for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")
                   for part, x in (("batch", 2048), ("token", 256), ("head", 64))}
        base = dict(strides, dtype=1, batch=2, q_len=3, kv_len=5, heads=4, kv_heads=2, head_dim=64, window=4,
                    sinks=1, lse=at, scratch=at,
                    **{n: at + 65536 * x for x, n in enumerate(("q", "k", "v", "out", "dout", "dq", "dk", "dv"))})
        return ctypes.byref(_lib.SparB200WindowAttention(**{**base, **k}))

    for bad in (dict(dtype=7), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(kv_heads=8),
                dict(head_dim=0), dict(head_dim=257), dict(window=0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(k=at + 1),
                dict(q_len=1 << 29), dict(kv_len=1 << 40), dict(batch=1 << 29, heads=64, kv_heads=64),
                dict(batch=1 << 12, kv_len=1 << 20), dict(scale=1e-31), dict(scale=1e31), dict(out_batch=0),
                dict(lse=at + 2), dict(lengths=at + 2), dict(first=at + 1)):
        assert lib.spar_b200_window_attention_forward(window(**bad), 0, None).code == 1, bad
        assert lib.spar_b200_window_attention_backward(window(**bad), 0, None).code == 1, bad
    for bad in (dict(out_token=0), dict(out_head=0), *(dict(out=at + 65536 * x) for x in range(3))):
        assert lib.spar_b200_window_attention_forward(window(**bad), 0, None).code == 1, bad
    written = {"dq": 5, "dk": 6, "dv": 7}
    for name, own in written.items():  # in the place of an input, or of another output
        for x in range(8):
            if x != own:
                bad = {name: at + 65536 * x}
                assert lib.spar_b200_window_attention_backward(window(**bad), 0, None).code == 1, bad
    for bad in (dict(dout=None), dict(lse=None), dict(dv=None), dict(scratch=None), dict(scratch=at + 16),
                dict(dq_token=0), dict(dk_head=0), dict(dv_batch=0)):
        assert lib.spar_b200_window_attention_backward(window(**bad), 0, None).code == 1, bad
    assert lib.spar_b200_window_attention_forward(window(batch=0, q=None, k=None), 0, None).code == 0
    assert lib.spar_b200_window_attention_forward(window(q_len=0, q=None, out=None), 0, None).code == 0
    assert lib.spar_b200_window_attention_backward(window(batch=0), 0, None).code == 0
    assert lib.spar_b200_window_attention_scratch_bytes(window(), 1, 0) >= 2 * 4 * 3 * 4
    for none in (dict(batch=0), dict(q_len=0), dict(kv_len=0), dict(q_len=0, kv_len=0)):
        for backward in (0, 1):  # no division by a count of zero
            assert lib.spar_b200_window_attention_scratch_bytes(window(**none), backward, 0) < 1 << 20
    # Partial sums stay within a quarter of a GB however many first tokens and rows there are.
    for size in (dict(sinks=4), dict(sinks=1 << 16), dict(sinks=1 << 16, batch=16), dict(sinks=1 << 16, window=1 << 20),
                 dict(sinks=200, heads=64, kv_heads=1, batch=1), dict(sinks=4, kv_len=130)):
        size = dict(q_len=1 << 16, kv_len=1 << 16) | size
        rows = size.get("batch", 2) * size.get("heads", 4) * size["q_len"] * 4
        got = lib.spar_b200_window_attention_scratch_bytes(window(**size), 1, 0)
        assert rows <= got <= rows + (1 << 28), (size, got)


def test_new_structures_mirror_the_header():
    """Sizes that a C compiler gives the header's structs (all members 8-byte aligned after the tags)."""
    from spar_b200 import _lib

    assert ctypes.sizeof(_lib.SparB200Rotary) == 352 == _lib.ROTARY.size
    assert ctypes.sizeof(_lib.SparB200WindowAttention) == 368 == _lib.WINDOW_ATTENTION.size
    for kind, packed in ((_lib.SparB200Rotary, _lib.ROTARY),
                         (_lib.SparB200WindowAttention, _lib.WINDOW_ATTENTION)):
        names = [name for name, _ in kind._fields_]
        held = kind.from_buffer_copy(packed.pack(*range(1, len(names) + 1)))
        assert [getattr(held, name) for name in names] == list(range(1, len(names) + 1))
    assert ctypes.sizeof(_lib.SparB200RotaryScaling) == 48
