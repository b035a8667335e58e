"""CPU: the causal and paged operators' structs, workspace sizes and refusals
(which come before anything touches a device)."""
import ctypes
import os
import subprocess

import pytest
import torch

import llmr_attn as L
from conftest import ROOT

HEADER = os.path.join(ROOT, "include", "llmr_attn.h")


@pytest.mark.parametrize("py_name,c_name", [("CausalDesc", "llmr_causal_desc"),
                                            ("PagedDesc", "llmr_paged_desc"),
                                            ("PlanDesc", "llmr_plan_desc"),
                                            ("PagedPrologueDesc", "llmr_paged_prologue_desc")])
def test_desc_layout_matches_c(py_name, c_name, tmp_path):
    cls = getattr(L, py_name)
    fields = [f[0] for f in cls._fields_]
    src = f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(){{printf("%zu\\n", sizeof({c_name}));'
    src += "".join(f'printf("%zu\\n", offsetof({c_name}, {f}));' for f in fields) + "return 0;}"
    c, exe = tmp_path / "t.c", tmp_path / "t"
    c.write_text(src)
    cc = "/usr/bin/gcc" if os.path.exists("/usr/bin/gcc") else "gcc"
    subprocess.run([cc, str(c), "-o", str(exe)], check=True)
    vals = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                           check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(cls)
    assert vals[1:] == [getattr(cls, f).offset for f in fields]


def test_workspace_is_zero_for_what_would_be_refused():
    def size(**kw):
        d = L.PagedDesc(**{**dict(n_seqs=2, total_tokens=9, max_q_len=5, n_heads=8, n_kv_heads=2,
                                  head_dim=128, dtype=L.F16, out_dtype=L.F16, scale=1.0,
                                  page_size=16, num_pages=10, max_pages=5), **kw})
        return L.lib.llmr_attention_paged_workspace_bytes(ctypes.byref(d))
    assert size() > 0
    for bad in (dict(head_dim=96), dict(n_heads=9), dict(n_kv_heads=0), dict(page_size=24),
                dict(page_size=8), dict(page_size=512), dict(num_pages=0), dict(num_pages=1 << 28),
                dict(dtype=L.F32), dict(out_dtype=7), dict(scale=0.0), dict(scale=float("nan")),
                dict(max_pages=0), dict(max_pages=1 << 27), dict(table_stride=4),
                dict(n_heads=258, n_kv_heads=2), dict(total_tokens=1 << 30)):
        assert size(**bad) == 0, bad
    assert L.lib.llmr_attention_paged_workspace_bytes(None) == 0
    with pytest.raises(L.LlmrError):
        L.attention_paged_workspace_bytes(n_seqs=1, total_tokens=1, max_q_len=1, n_heads=3,
                                          n_kv_heads=2, head_dim=64)


def test_null_context_is_refused():
    for name, args in (("llmr_attention_causal", 7), ("llmr_attention_paged", 9),
                       ("llmr_paged_plan", 11), ("llmr_paged_prologue", 13)):
        assert getattr(L.lib, name)(None, *[None] * args) == L.EINVAL


class NoDevice:
    """Stands for a context; the library must not be reached with it. -1 is
    where torch says that host tensors are."""
    handle = None

    def __init__(self, device=-1):
        self.device = device

    def check(self, rc):
        raise AssertionError("a refused call reached the library")


B = torch.bfloat16


def z(*shape, dtype=B):
    return torch.zeros(shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def refused(f, word=""):
    with pytest.raises(L.LlmrError) as e:
        f()
    assert e.value.status == L.EINVAL and word in str(e.value), e.value


@pytest.mark.parametrize("change,word", [
    (dict(q=z(5, 4, 96)), "head_dim"), (dict(q=z(5, 5, 64)), "multiple"), (dict(q=z(5, 256)), "q must"),
    (dict(q=z(5, 4, 64, dtype=torch.float32)), "dtype"), (dict(k=z(5, 2, 64, dtype=torch.float16)), "dtype"),
    (dict(k=z(4, 2, 64)), "k is"), (dict(v=z(5, 1, 64)), "v is"), (dict(o=z(5, 4, 128)), "o is"),
    (dict(o=z(5, 255)), "o must"), (dict(v=z(5, 64, 2).transpose(1, 2)), "dense"),
    (dict(cu=torch.zeros(2, dtype=torch.int64)), "int32"), (dict(cu=i32(4)[::2]), "dense"),
    (dict(cu=i32(0)), "cu_seqlens"), (dict(lse=z(4, 5)), "lse"), (dict(lse=z(5, 4, dtype=torch.float32)), "lse"),
    (dict(), "cuda:0"),
])
def test_causal_refuses(change, word):
    a = {**dict(q=z(5, 4, 64), k=z(5, 2, 64), v=z(5, 2, 64), o=z(5, 4, 64), cu=i32(2), lse=None), **change}
    refused(lambda: L.attention_causal(NoDevice(0 if not change else -1), a["q"], a["k"], a["v"], a["o"], a["cu"], scale=0.1,
                                       lse=a["lse"]), word)


def test_broadcast_inputs_are_refused():
    refused(lambda: L._step(2, z(5, 1, 64).expand(5, 2, 64).stride(1)), "broadcast")
    assert L._step(1, 0) == 0 and L._step(5, 128) == 128


@pytest.mark.parametrize("change,word", [
    (dict(kc=z(3, 16, 64)), "k_cache"), (dict(vc=z(3, 32, 2, 64)), "v_cache"),
    (dict(kc=z(3, 16, 2, 64, dtype=torch.float16)), "dtype"), (dict(kc=z(3, 16, 3, 64)), "multiple"),
    (dict(vc=z(3, 16, 2, 64, dtype=torch.float16)), "dtype"),
    (dict(cu=i32(4)), "cu_q"), (dict(kv=torch.zeros(2, dtype=torch.int64)), "kv_lens"),
    (dict(table=i32(3, 4)), "block_table"), (dict(table=i32(2, 0)), "block_table"),
    (dict(table=i32(2, 8)[:, ::2]), "block_table"), (dict(max_q=-1), "max_q_len"), (dict(), "cuda:0"),
])
def test_paged_refuses(change, word):
    a = {**dict(q=z(5, 4, 64), kc=z(3, 16, 2, 64), vc=z(3, 16, 2, 64), o=z(5, 4, 64), cu=i32(3), kv=i32(2),
                table=i32(2, 4), max_q=5), **change}
    refused(lambda: L.attention_paged(NoDevice(0 if not change else -1), a["q"], a["kc"], a["vc"], a["o"], a["cu"], a["kv"],
                                      a["table"], scale=0.1, max_q_len=a["max_q"]), word)


@pytest.mark.parametrize("change,word", [
    (dict(new=i32(4)), "new_lens"), (dict(cu=i32(3)), "cu_q"), (dict(slots=i32(8)), "slots"),
    (dict(kv=i32(2)), "kv_lens"), (dict(n_free=i32(2)), "n_free"), (dict(table=i32(2, 4)), "block_table"),
    (dict(free=torch.zeros(5, dtype=torch.int64)), "free_pages"), (dict(page=0), "page_size"),
    (dict(), "cuda:0"),
])
def test_plan_refuses(change, word):
    a = {**dict(ctx=i32(3), new=i32(3), free=i32(5), n_free=i32(1), table=i32(3, 4), cu=i32(4), kv=i32(3),
                pos=i32(9), slots=i32(9), out=i32(1), page=16), **change}
    refused(lambda: L.paged_plan(NoDevice(0 if not change else -1), a["ctx"], a["new"], a["free"], a["n_free"], a["table"], a["cu"],
                                 a["kv"], a["pos"], a["slots"], a["out"], page_size=a["page"]), word)


F = torch.float32


@pytest.mark.parametrize("change,word", [
    (dict(k=z(5, 3, 64)), "k_cache"), (dict(v=z(5, 2, 64, dtype=F)), "dtype"), (dict(q_out=None), "together"),
    (dict(q_out=z(5, 4, 64, dtype=F)), "dtype"), (dict(kc=z(3, 16, 2, 64, dtype=F)), "caches"),
    (dict(slots=i32(4)), "slots"), (dict(pos=i32(6)), "positions"), (dict(pos=None), "positions"),
    (dict(sin=None), "together"), (dict(cos=z(9, 64, dtype=F)), "cos"), (dict(cos=None, sin=None), "half"),
    (dict(q_gain=z(64)), "q_gain"), (dict(k_gain=z(65, dtype=F)), "k_gain"),
    (dict(q=None, q_out=None), "q_gain"), (dict(), "cuda:0"),
])
def test_prologue_refuses(change, word):
    a = {**dict(q=z(5, 4, 64), k=z(5, 2, 64), v=z(5, 2, 64), q_out=z(5, 4, 64), kc=z(3, 16, 2, 64),
                vc=z(3, 16, 2, 64), pos=i32(5), slots=i32(5), cos=z(9, 32, dtype=F), sin=z(9, 32, dtype=F),
                q_gain=z(64, dtype=F), k_gain=None), **change}
    refused(lambda: L.paged_prologue(NoDevice(0 if not change else -1), a["q"], a["k"], a["v"], a["q_out"], a["kc"], a["vc"], a["pos"],
                                     a["slots"], q_gain=a["q_gain"], k_gain=a["k_gain"], cos=a["cos"],
                                     sin=a["sin"], half=True), word)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_the_longest_context(page):
    """Lengths of more than 2^31 - 256 keys are refused: rounded up to a block of 128 they pass an int."""
    def size(max_pages):
        d = L.PagedDesc(n_seqs=1, total_tokens=1, max_q_len=1, n_heads=4, n_kv_heads=1, head_dim=64,
                        dtype=L.F16, out_dtype=L.F16, scale=1.0, page_size=page, num_pages=4,
                        max_pages=max_pages)
        return L.lib.llmr_attention_paged_workspace_bytes(ctypes.byref(d))
    most = (2 ** 31 - 256) // page
    assert size(most) > 0 and size(most + 1) == 0
