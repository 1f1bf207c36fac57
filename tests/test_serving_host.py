"""The serving entry points on the host: refusals that need no GPU, and the
binding's structures against the header's."""
import ctypes
import re

from conftest import ROOT


def test_null_contexts_are_refused():
    import tier_b200 as tk
    from tier_b200 import build
    build.build()
    lib = tk.load()
    c, s = tk.KvCache(), tk.Seqs()
    p, q = ctypes.byref(c), ctypes.byref(s)
    for st in (lib.tk_kv_append(None, p, q, None, None, 0, 0, 0, None), lib.tk_kv_read(None, p, q, None, None, 0, 0, 0, None),
               lib.tk_kv_attend(None, p, q, None, 0, 0, 4, 1.0, 0, None, 0, None),
               lib.tk_draft_verify(None, 1, None, 1, 10, None, 10, None, 0, None, None, None, 1.0, None, None, None, None)):
        assert st == tk.TK_ERR_INVALID and b"null context" in lib.tk_last_error_string()


def test_structures_match_the_header():
    import tier_b200 as tk
    text = (ROOT / "include" / "tierk.h").read_text()
    for name, cls in (("tk_kvcache", tk.KvCache), ("tk_seqs", tk.Seqs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        fields = []
        for decl in body.split(";"):
            m = re.match(r"\s*(?:const\s+)?(int32_t|int|void)\s+(.*)", decl.strip(), re.S)
            if m:
                fields += [(f.strip().lstrip("*"), "*" in f) for f in m.group(2).split(",")]
        assert [f for f, _ in fields] == [f for f, _ in cls._fields_]
        assert [ctypes.c_void_p if ptr else ctypes.c_int for _, ptr in fields] == [t for _, t in cls._fields_]


def test_references_agree_with_themselves():
    """Packing and unpacking invert each other, and every value n * d is exact in fp16."""
    import numpy as np
    import kv_ref as ref
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 2, 128)) * np.exp(rng.uniform(-8, 8, (50, 2, 1)))).astype(np.float32)
    n, d = ref.quantize(x)
    back = ref.unpack(ref.pack(n), d)
    assert np.array_equal(back, n * np.repeat(d.astype(np.float64), 32, -1))
    assert np.array_equal(back, back.astype(np.float16).astype(np.float64))
    step = np.repeat(np.abs(x.reshape(50, 2, 4, 32)).max(-1) / 8, 32, -1)
    assert (np.abs(back - x) <= step * (1 + 2.0 ** -5)).all()
