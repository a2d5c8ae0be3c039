"""CPU tests of the serving operators' boundary: what the C entry points refuse without a context, and the argument checks of
the Python binding, run against a stand-in for the library (nothing is launched)."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

import vknn_b200
from vknn_b200 import capi


class Recorder:
    """Stands in for the loaded library: notes the calls and their argument structs, and succeeds."""

    STRUCTS = {"vkc_attn_prefill_packed": capi.PACKED_ARGS, "vkc_kv_append_q8": capi.APPEND_ARGS, "vkc_attn_decode_q8": capi.DECODE_Q8_ARGS}

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        s = self.STRUCTS[name]
        return lambda h, args, stream: self.calls.append((name, s.unpack(args))) or 0


@pytest.fixture
def fake():
    c = vknn_b200.Context.__new__(vknn_b200.Context)
    c.lib, c.h, c.device = Recorder(), None, -1  # -1 is what CPU tensors answer for their device
    c._stream = lambda stream: None
    return c


def z(*s, dt=torch.float16):
    return torch.zeros(*s, dtype=dt)


def cache(b=2, hkv=2, lmax=64, d=64, block=32, dt=torch.float8_e4m3fn):
    return z(b, hkv, lmax, d, dt=dt), z(b, hkv, lmax, d, dt=dt), z(b, hkv, lmax // block, dt=torch.float32), z(b, hkv, lmax // block, dt=torch.float32)


def test_the_current_stream_with_and_without_torchs_private_function(monkeypatch):
    c = vknn_b200.Context.__new__(vknn_b200.Context)
    c.h, c.device = None, 3
    seen = []
    for handle, want in ((0x1234, 0x1234), (0, 1)):  # 0, the legacy stream, goes by its explicit handle
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: seen.append(d) or handle, raising=False)
        assert c._stream(None).value == want
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream")
        monkeypatch.setattr(torch.cuda, "current_stream", lambda d: seen.append(d) or type("S", (), {"cuda_stream": handle}))
        assert c._stream(None).value == want
    assert seen == [3] * 4 and c._stream(77).value == 77


def test_null_context_is_refused():
    lib = vknn_b200.load_library()
    args = C.create_string_buffer(256)
    for f in (lib.vkc_attn_prefill_packed, lib.vkc_kv_append_q8, lib.vkc_attn_decode_q8):
        assert f(None, C.addressof(args), None) == -1 and f(None, None, None) == -1
    assert lib.vkc_attn_decode_q8_workspace_bytes(0, 1, 1, 32, 64) == 0 and lib.vkc_attn_decode_q8_workspace_bytes(2, 8, 2, 4096, 128) > 0


def test_lengths_of_a_single_sequence_may_come_from_a_column(fake):
    k, v, ks, vs = cache(b=1)
    lens = z(3, 2, dt=torch.int32)[:1, 1]
    fake.kv_append_q8(z(1, 2, 64), z(1, 2, 64), k, v, ks, vs, kv_len=lens)
    assert fake.lib.calls[0][1][13] == lens.data_ptr()
    with pytest.raises(ValueError):
        fake.kv_append_q8(z(2, 2, 64), z(2, 2, 64), *cache(), kv_len=z(2, 2, dt=torch.int32)[:, 1])


def test_argument_structs_have_the_layout_of_the_c_compiler(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    # every field gets its own number (the floats and ints too), packed by Python and read by C
    fields = {"attn_prefill_packed": (capi.PACKED_ARGS, "Q K V O nseq Hq Hkv D total_q total_k cu_q cu_k q_strides[0] q_strides[1] k_strides[0] k_strides[1] "
                                      "v_strides[0] v_strides[1] o_strides[0] o_strides[1] scale causal dtype"),
              "kv_append_q8": (capi.APPEND_ARGS, "K V Kc Vc k_scale v_scale B Hkv Lmax D block total cu kv_len k_strides[0] k_strides[1] v_strides[0] v_strides[1] "
                               "dtype cache_dtype"),
              "attn_decode_q8": (capi.DECODE_Q8_ARGS, "Q Kc Vc k_scale v_scale O B Hq Hkv Lmax D block kv_len workspace workspace_bytes scale dtype cache_dtype")}
    body = ""
    for name, (s, text) in fields.items():
        names = text.split()
        (tmp_path / name).write_bytes(s.pack(*(float(i + 1) if n == "scale" else i + 1 for i, n in enumerate(names))) + bytes(16))
        body += ('{ vkc_%s_args a; FILE *f = fopen("%s", "rb"); if (!f || fread(&a, 1, sizeof a, f) != sizeof a) return 1; fclose(f); long long v[] = {%s}; '
                 'for (int i = 0; i < %d; ++i) if (v[i] != i + 1) { printf("%s %%d %%lld\\n", i, v[i]); return 2; } }\n'
                 % (name, tmp_path / name, ", ".join("(long long)%s a.%s" % ("" if n == "scale" else "(intptr_t)", n) for n in names), len(names), name))
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text('#include <stdio.h>\n#include <stdint.h>\n#include "vknn_cuda.h"\nint main(void) {\n%s return 0; }\n' % body)
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", inc, str(src), "-o", str(exe)])
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "" and subprocess.call([str(exe)]) == 0


def test_packed_arguments_reach_the_library_as_given(fake):
    qkv, o, cu = z(10, 8, 64), z(10, 4, 64), z(3, dt=torch.int32)
    fake.attn_prefill_packed(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], o, 0.5, cu, causal=False)
    (name, a), = fake.lib.calls
    assert name == "vkc_attn_prefill_packed" and a[4:10] == (2, 4, 2, 64, 10, 10) and a[10:12] == (cu.data_ptr(), 0)
    assert a[12:20] == (512, 64) * 3 + (256, 64) and a[20:] == (0.5, 0, vknn_b200.F16)


def test_cache_arguments_reach_the_library_as_given(fake):
    c = cache(b=3, lmax=128, block=32, dt=torch.int8)
    lens = z(3, dt=torch.int32)
    fake.kv_append_q8(z(3, 2, 64), z(3, 2, 64), *c, lens)
    fake.attn_decode_q8(z(3, 6, 64), *c, z(3, 6, 64), 0.25, kv_len=lens)
    (n1, a), (n2, b) = fake.lib.calls
    assert n1 == "vkc_kv_append_q8" and a[6:14] == (3, 2, 128, 64, 32, 3, 0, lens.data_ptr()) and a[14:] == (128, 64, 128, 64, vknn_b200.F16, vknn_b200.I8)
    assert n2 == "vkc_attn_decode_q8" and b[6:] == (3, 6, 2, 128, 64, 32, lens.data_ptr(), 0, 0, 0.25, vknn_b200.F16, vknn_b200.I8)


def test_packed_refusals(fake):
    q, kv, lens = z(6, 4, 64), z(6, 2, 64), z(2, dt=torch.int32)
    for args, more in (((q, kv, kv, q, 1.0, lens.long()), {}), ((q, kv, kv[:5], q, 1.0, lens), {}), ((q, kv.float(), kv, q, 1.0, lens), {}),
                       ((q, kv, kv, q[:5], 1.0, lens), {}), ((q, kv, kv, q, 1.0, lens), {"cu_k": lens[:1]}), ((q, z(6, 2, 32), z(6, 2, 32), q, 1.0, lens), {}),
                       ((q.transpose(0, 2), kv, kv, q.transpose(0, 2), 1.0, lens), {})):
        with pytest.raises(ValueError):
            fake.attn_prefill_packed(*args, **more)
    wide = z(1, 1, 64)
    for args in ((q, wide.expand(6, 2, 64), kv, q), (q, kv, wide.expand(6, 2, 64), q), (wide.expand(6, 4, 64), kv, kv, q)):
        with pytest.raises(ValueError):
            fake.attn_prefill_packed(*args, 1.0, lens)
    assert not fake.lib.calls
    fake.attn_prefill_packed(q, z(6, 1, 64).expand(6, 2, 64), kv, q, 1.0, lens)  # one head for all is an ordinary stride
    assert fake.lib.calls[0][1][14:16] == (64, 0)


def test_append_refusals(fake):
    k, lens = z(2, 2, 64), z(2, dt=torch.int32)
    kc, vc, ks, vs = cache()
    for args in ((k, k, kc, vc, ks[..., :1], vs, lens), (k, k, kc, vc[:1], ks, vs, lens), (k, k, kc, vc.view(torch.int8), ks, vs, lens),
                 (k, k, kc.half(), vc.half(), ks, vs, lens), (k, k, kc, vc, ks.half(), vs.half(), lens), (k, k[:1], kc, vc, ks, vs, lens),
                 (z(2, 4, 64), z(2, 4, 64), kc, vc, ks, vs, lens), (k, k.float(), kc, vc, ks, vs, lens), (k, k, kc, vc, ks, vs, lens.long()),
                 (k, k, kc, vc, ks, vs, lens[:1]), (k, k, kc, vc, z(2, 2, 3, dt=torch.float32), z(2, 2, 3, dt=torch.float32), lens),
                 (k, k, kc.transpose(0, 1), vc.transpose(0, 1), ks, vs, lens)):
        with pytest.raises(ValueError):
            fake.kv_append_q8(*args)
    with pytest.raises(ValueError):
        fake.kv_append_q8(k, k, kc, vc, ks, vs, lens, cu=lens)  # three offsets are wanted
    with pytest.raises(ValueError):
        fake.kv_append_q8(z(1, 1, 64).expand(2, 2, 64), k, kc, vc, ks, vs, lens)
    assert not fake.lib.calls


def test_decode_refusals(fake):
    q, lens, c = z(2, 4, 64), z(2, dt=torch.int32), cache()
    for args in ((z(3, 4, 64), *c, z(3, 4, 64), 1.0), (q, *c, q.bfloat16(), 1.0), (q, *c, z(2, 2, 64), 1.0), (q.transpose(0, 1).contiguous().transpose(0, 1), *c, q, 1.0),
                 (z(2, 4, 128), *c, z(2, 4, 128), 1.0)):
        with pytest.raises(ValueError):
            fake.attn_decode_q8(*args, kv_len=lens)
    with pytest.raises(ValueError):
        fake.attn_decode_q8(q, *c, z(2, 4, 64), 1.0, kv_len=lens.float())
    with pytest.raises(ValueError):
        fake.attn_decode_q8(q, *c, z(2, 4, 64), 1.0, kv_len=lens, workspace=z(64, 64).t()[::2])
    fake.device = 0  # tensors that lie somewhere else
    with pytest.raises(ValueError):
        fake.attn_decode_q8(q, *c, z(2, 4, 64), 1.0, kv_len=lens)
    assert not fake.lib.calls


def test_argument_structs_are_as_long_as_the_c_compilers(tmp_path):
    """The library copies its argument struct whole, the padding at its end included."""
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    structs = {"attn_prefill_packed": capi.PACKED_ARGS, "kv_append_q8": capi.APPEND_ARGS, "attn_decode_q8": capi.DECODE_Q8_ARGS}
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text('#include <stdio.h>\n#include "vknn_cuda.h"\nint main(void) {\n%s return 0; }\n' %
                   "".join('printf("%s %%d\\n", (int) sizeof(vkc_%s_args));\n' % (n, n) for n in structs))
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", inc, str(src), "-o", str(exe)])
    sizes = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    assert {n: int(x) for n, x in sizes.items()} == {n: s.size for n, s in structs.items()}
    for s in structs.values():
        assert s.size % s.__class__("@P").size == 0
