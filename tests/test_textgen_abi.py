"""The text-generation calls' checks of their arguments, without a GPU: every
refusal comes before any device call, as a code and a message."""
import ctypes

import numpy as np
import pytest


@pytest.fixture()
def structs(pkg):
    import importlib

    tg = importlib.import_module("bark3_b200.textgen")
    buf = np.zeros(64, np.float32)
    p = (buf.ctypes.data + 15) // 16 * 16
    cache = tg._Cache(p, p, p, p, None, 4, 2, 16, 64)
    batch = tg._Batch(p, p, p, 3, 3, 1, 1)
    app = tg._Append(p, p, p, p, 256, 64, 128, 64, 128, 64, None, None, None, None, None, 1e-6, pkg.DTYPE_F16,
                     pkg.DTYPE_F16, 4, 0, 0, 0)
    att = tg._Attend(p, p, None, 256, 64, 0.125, pkg.DTYPE_F16, 4, 1, 1, 0)
    smp = tg._Sample(p, p, None, None, None, None, p, None, 10, pkg.DTYPE_F32, 1, 10)
    return p, cache, batch, app, att, smp, buf


def ref(x):
    return ctypes.byref(x) if x is not None else None


def test_struct_layouts_match_the_header(pkg, tmp_path):
    """sizeof and field offsets as a C compiler sees them."""
    import importlib
    import subprocess

    tg = importlib.import_module("bark3_b200.textgen")
    pairs = [("b3_kv_cache", tg._Cache), ("b3_kv_batch", tg._Batch), ("b3_kv_append_args", tg._Append),
             ("b3_kv_attend_args", tg._Attend), ("b3_sample_args", tg._Sample)]
    lines, want = [], []
    for name, s in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(s))
        for f in s._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f[0]}));')
            want.append(getattr(s, f[0]).offset)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{pkg.HEADER}"\nint main(void) {{ '
                   + " ".join(lines) + " return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want
    assert f"B3_SAMPLE_MAX_VOCAB {tg.SAMPLE_MAX_VOCAB}" in pkg.HEADER.read_text()


def test_cache_and_batch_are_checked(pkg, structs):
    p, cache, batch, app, att, smp, _ = structs
    L = pkg.lib()
    for obj, field, value, text in (
            (cache, "k", None, "null buffer"), (cache, "v_scale", None, "null buffer"), (cache, "head_dim", 96, "head_dim"),
            (cache, "page_tokens", 48, "page_tokens"), (cache, "page_tokens", 0, "page_tokens"),
            (cache, "pages", 0, "cache of"), (cache, "pages", 1 << 27, "cache of"), (cache, "kv_heads", 0, "cache of"),
            (cache, "v", p + 4, "16-byte"), (batch, "cu_q", None, "null buffer"), (batch, "page_table", None, "null buffer"),
            (batch, "n_seq", 0, "batch of"), (batch, "tokens", -1, "batch of"), (batch, "table_stride", 2, "batch of"),
            (batch, "table_width", 0, "batch of")):
        old = getattr(obj, field)
        setattr(obj, field, value)
        for rc in (L.b3_kv_append(ref(cache), ref(batch), ref(app), None),
                   L.b3_kv_attend(ref(cache), ref(batch), ref(att), None, 0, None),
                   L.b3_kv_attend_workspace(ref(cache), ref(batch), ref(att))):
            assert rc == pkg.B3_EINVAL and text in pkg.last_error(), (field, value)
        setattr(obj, field, old)
    for a, b, c in ((None, batch, app), (cache, None, app), (cache, batch, None)):
        assert L.b3_kv_append(ref(a), ref(b), ref(c), None) == pkg.B3_EINVAL
    for a, b, c in ((None, batch, att), (cache, None, att), (cache, batch, None)):
        assert L.b3_kv_attend(ref(a), ref(b), ref(c), None, 0, None) == pkg.B3_EINVAL
        assert L.b3_kv_attend_workspace(ref(a), ref(b), ref(c)) == pkg.B3_EINVAL


def test_append_attend_and_sample_are_checked(pkg, structs):
    p, cache, batch, app, att, smp, _ = structs
    L = pkg.lib()
    for field, value, text in (("q", None, "null"), ("q_out", None, "null"), ("q_out", p + 8, "16-byte"),
                               ("q_heads", 3, "multiple"), ("q_heads", 0, "multiple"), ("dtype", 7, "dtype"),
                               ("out_dtype", pkg.DTYPE_F32, "out_dtype"), ("k_norm", p + 4, "16-byte"), ("cos", p, "together")):
        old = getattr(app, field)
        setattr(app, field, value)
        assert L.b3_kv_append(ref(cache), ref(batch), ref(app), None) == pkg.B3_EINVAL and text in pkg.last_error(), field
        setattr(app, field, old)
    app.cos, app.sin, app.rot_rows = p, p, 4
    for rot in (0, 8, 24, 80, -16):
        app.rot_dim = rot
        assert L.b3_kv_append(ref(cache), ref(batch), ref(app), None) == pkg.B3_EINVAL and "rot_dim" in pkg.last_error()
    for field, value, text in (("q", None, "null"), ("out", p + 2, "16-byte"), ("q_heads", 5, "multiple"),
                               ("dtype", pkg.DTYPE_F32, "dtype"), ("max_q", 0, "max_q"), ("window", -3, "window")):
        old = getattr(att, field)
        setattr(att, field, value)
        assert L.b3_kv_attend(ref(cache), ref(batch), ref(att), None, 0, None) == pkg.B3_EINVAL
        assert text in pkg.last_error(), field
        setattr(att, field, old)
    att.causal, att.window = 0, 8
    assert L.b3_kv_attend(ref(cache), ref(batch), ref(att), None, 0, None) == pkg.B3_EINVAL
    for field, value in (("logits", None), ("uniform", None), ("ids", None), ("rows", -1), ("vocab", 0),
                         ("vocab", 262145), ("row_stride", 9), ("dtype", 5)):
        old = getattr(smp, field)
        setattr(smp, field, value)
        assert L.b3_sample(ref(smp), None) == pkg.B3_EINVAL, field
        setattr(smp, field, old)
    assert L.b3_sample(None, None) == pkg.B3_EINVAL
    smp.rows = 0
    assert L.b3_sample(ref(smp), None) == 0


def test_a_sequence_of_nearly_two_to_the_31_tokens_is_refused(pkg, structs):
    """Past 2^31 - 1024 tokens a place rounded up to a kernel's block would leave 32 bits."""
    p, cache, batch, app, att, smp, _ = structs
    L = pkg.lib()
    batch.table_width = batch.table_stride = (1 << 31) // cache.page_tokens - 63
    for rc in (L.b3_kv_append(ref(cache), ref(batch), ref(app), None),
               L.b3_kv_attend(ref(cache), ref(batch), ref(att), None, 0, None),
               L.b3_kv_attend_workspace(ref(cache), ref(batch), ref(att))):
        assert rc == pkg.B3_EINVAL and "2147482624 tokens" in pkg.last_error()
