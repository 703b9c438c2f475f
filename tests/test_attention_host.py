"""The entry points of csrc/attention.cpp on the CPU: what they refuse, before any launch,
and what they do with scratch, over a HIP runtime and launchers that only keep books."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import smoe_amd
from smoe_amd import SMOE_ERR_ARG, SMOE_ERR_CAPTURE, SMOE_ERR_HIP, SMOE_ERR_SHAPE, SMOE_OK

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = 1 << 20        # stands for any device address


@pytest.fixture(scope="module")
def so(tmp_path_factory):
    cxx = "/opt/rocm/llvm/bin/clang++"
    cxx = cxx if os.path.exists(cxx) else shutil.which("clang++")
    out = str(tmp_path_factory.mktemp("fake") / "libattention_fake.so")
    src = os.path.join(ROOT, "s-moe_amd", "csrc")
    r = subprocess.run(
        [cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
         "-I" + os.path.join(ROOT, "include"), "-I" + src, os.path.join(src, "bridge.cpp"),
         os.path.join(src, "attention.cpp"), os.path.join(ROOT, "tests", "fake_hip.cpp"),
         os.path.join(ROOT, "tests", "fake_attention.cpp"), "-Wl,-Bsymbolic", "-o", out],
        capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return out


class Lib:
    def __init__(self, so):
        self.lib = C.CDLL(so)
        for name, res, args in smoe_amd.SIGNATURES:
            if hasattr(self.lib, name):
                getattr(self.lib, name).restype, getattr(self.lib, name).argtypes = res, args
        self.lib.fake_attention.restype, self.lib.fake_attention.argtypes = C.c_uint64, [C.c_char_p]
        self.lib.fake_count.restype, self.lib.fake_count.argtypes = C.c_uint64, [C.c_char_p]
        self.lib.fake_budget.argtypes = [C.c_size_t]
        self.lib.fake_is_live.argtypes = [C.c_uint64]
        self.lib.fake_budget(C.c_size_t(-1).value)
        self.lib.fake_capturing(0)
        self.ctx = self.lib.smoe_metal_init(1 << 15)
        assert self.ctx

    def close(self):
        self.lib.fake_capturing(0)
        self.lib.smoe_metal_destroy(self.ctx)
        assert self.lib.fake_count(b"allocations") == 0       # all given back

    def booked(self, what="launches"):
        return self.lib.fake_attention(what.encode())

    def call(self, name, *args):
        n = self.booked()
        rc = getattr(self.lib, "smoe_hip_" + name)(self.ctx, *[C.byref(a) if a is not None else None for a in args])
        assert (self.booked() == n + 1) == (rc == SMOE_OK), "a refused call launches nothing"
        if rc != SMOE_OK:
            assert self.lib.smoe_hip_last_error(self.ctx)
        return rc


@pytest.fixture
def lib(so):
    b = Lib(so)
    yield b
    b.close()


def qk(**more):
    a = dict(q=DEV, q_out=DEV, k=DEV, k_out=DEV, q_norm_w=DEV, k_norm_w=DEV, rope_cos=DEV, rope_sin=DEV, positions=DEV,
             q_stride=4096, q_out_stride=4096, k_stride=512, k_out_stride=512, n_rows=7, n_positions=100, num_heads=32,
             num_kv_heads=4, head_dim=128, type=smoe_amd.TYPE_BF16)
    a.update(more)
    return smoe_amd.SmoeQkRowsArgs(**a)


def prompt(**more):
    a = dict(q=DEV, k=DEV, v=DEV, out=DEV, q_offsets=DEV, k_offsets=DEV, q_stride=4096, k_stride=512, v_stride=512,
             out_stride=4096, n_seqs=2, q_rows=10, k_rows=10, max_k=10, num_heads=32, num_kv_heads=4, head_dim=128,
             type=smoe_amd.TYPE_F16, scale=0.1)
    a.update(more)
    return smoe_amd.SmoePromptAttnArgs(**a)


def cache(**more):
    a = dict(k_codes=DEV, v_codes=DEV, k_params=DEV, v_params=DEV, n_slots=3, capacity=100, num_kv_heads=4, head_dim=128)
    a.update(more)
    return smoe_amd.SmoeKv4Cache(**a)


def rows(**more):
    a = dict(k=DEV, v=DEV, offsets=DEV, slots=DEV, start=DEV, lens_out=None, k_stride=512, v_stride=512, n_seqs=2,
             n_rows=10, type=smoe_amd.TYPE_F32)
    a.update(more)
    return smoe_amd.SmoeKv4RowsArgs(**a)


def attn(**more):
    a = dict(q=DEV, out=DEV, slots=DEV, lens=DEV, q_stride=4096, out_stride=4096, n_seqs=2, max_len=10, num_heads=32,
             type=smoe_amd.TYPE_F32, scale=0.1)
    a.update(more)
    return smoe_amd.SmoeKv4AttnArgs(**a)


@pytest.mark.parametrize("more,rc", [
    ({}, SMOE_OK), (dict(q_norm_w=None, k_norm_w=None), SMOE_OK), (dict(rope_cos=None, rope_sin=None, positions=None), SMOE_OK),
    (dict(k=None, k_out=None), SMOE_OK), (dict(q=None, q_out=None), SMOE_OK),
    (dict(q=None, q_out=None, k=None, k_out=None), SMOE_ERR_ARG), (dict(q_out=None), SMOE_ERR_ARG),
    (dict(k=None), SMOE_ERR_ARG), (dict(rope_sin=None), SMOE_ERR_ARG), (dict(positions=None), SMOE_ERR_ARG),
    (dict(n_positions=0), SMOE_ERR_ARG), (dict(type=3), SMOE_ERR_ARG), (dict(head_dim=96), SMOE_ERR_SHAPE),
    (dict(num_heads=0), SMOE_ERR_ARG), (dict(num_heads=1025, q_stride=1 << 20, q_out_stride=1 << 20), SMOE_ERR_SHAPE),
    (dict(q=DEV + 8), SMOE_ERR_SHAPE), (dict(q_stride=4095), SMOE_ERR_SHAPE), (dict(q_stride=4100), SMOE_ERR_SHAPE),
    (dict(k_out_stride=1 << 23), SMOE_ERR_SHAPE), (dict(rope_cos=DEV + 4), SMOE_ERR_ARG),
    (dict(n_rows=1 << 26), SMOE_ERR_SHAPE),
])
def test_qk_rows(lib, more, rc):
    assert lib.call("qk_norm_rope", qk(**more)) == rc


@pytest.mark.parametrize("more,rc", [
    ({}, SMOE_OK), (dict(k_offsets=None), SMOE_OK), (dict(max_k=0), SMOE_OK), (dict(k_rows=0, k=None, v=None), SMOE_OK),
    (dict(q=None), SMOE_ERR_ARG), (dict(out=None), SMOE_ERR_ARG), (dict(v=None), SMOE_ERR_ARG),
    (dict(q_offsets=None), SMOE_ERR_ARG), (dict(n_seqs=0), SMOE_ERR_ARG), (dict(type=7), SMOE_ERR_ARG),
    (dict(scale=0.0), SMOE_ERR_ARG), (dict(scale=-1.0), SMOE_ERR_ARG), (dict(scale=float("nan")), SMOE_ERR_ARG),
    (dict(scale=float("inf")), SMOE_ERR_ARG), (dict(head_dim=32), SMOE_ERR_SHAPE), (dict(num_heads=30), SMOE_ERR_SHAPE),
    (dict(num_kv_heads=0), SMOE_ERR_SHAPE), (dict(v=DEV + 2), SMOE_ERR_SHAPE), (dict(k_stride=508), SMOE_ERR_SHAPE),
    (dict(out_stride=4097), SMOE_ERR_SHAPE), (dict(v_stride=(1 << 22) + 8), SMOE_ERR_SHAPE),
    (dict(q_rows=1 << 26), SMOE_ERR_SHAPE), (dict(k_rows=1 << 31), SMOE_ERR_SHAPE), (dict(n_seqs=1 << 30), SMOE_ERR_SHAPE),
])
def test_prompt(lib, more, rc):
    assert lib.call("attention_prompt", prompt(**more)) == rc


CACHES = [(dict(k_codes=None), SMOE_ERR_ARG), (dict(v_params=None), SMOE_ERR_ARG), (dict(n_slots=0), SMOE_ERR_ARG),
          (dict(capacity=0), SMOE_ERR_ARG), (dict(num_kv_heads=0), SMOE_ERR_ARG), (dict(head_dim=80), SMOE_ERR_SHAPE),
          (dict(v_codes=DEV + 8), SMOE_ERR_ARG), (dict(capacity=(1 << 24) + 1), SMOE_ERR_SHAPE),
          (dict(n_slots=1 << 31), SMOE_ERR_SHAPE)]


@pytest.mark.parametrize("more,rc", CACHES)
def test_caches(lib, more, rc):
    assert lib.call("kv4_append", cache(**more), rows()) == rc
    assert lib.call("kv4_read", cache(**more), rows()) == rc
    assert lib.call("attention_kv4", cache(**more), attn()) == rc


@pytest.mark.parametrize("more,rc", [
    ({}, SMOE_OK), (dict(slots=None), SMOE_OK), (dict(offsets=None, n_rows=2), SMOE_OK),
    (dict(offsets=None), SMOE_ERR_ARG), (dict(k=None), SMOE_ERR_ARG), (dict(start=None), SMOE_ERR_ARG),
    (dict(n_seqs=0), SMOE_ERR_ARG), (dict(type=3), SMOE_ERR_ARG), (dict(v=DEV + 4), SMOE_ERR_SHAPE),
    (dict(k_stride=511), SMOE_ERR_SHAPE), (dict(v_stride=514), SMOE_ERR_SHAPE), (dict(n_rows=1 << 28), SMOE_ERR_SHAPE),
])
def test_cache_rows(lib, more, rc):
    assert lib.call("kv4_append", cache(), rows(**more)) == rc
    assert lib.call("kv4_read", cache(), rows(**more)) == rc


def test_the_largest_calls(lib):
    """A launch has less than 2^32 threads; what would need more is refused, not left to the launch."""
    one = dict(num_heads=1, num_kv_heads=1)
    for n, rc in (((1 << 26) - 4, SMOE_OK), ((1 << 26) - 3, SMOE_ERR_SHAPE)):
        assert lib.call("qk_norm_rope", qk(n_rows=n, **one)) == rc
        for name in ("kv4_append", "kv4_read"):
            assert lib.call(name, cache(num_kv_heads=1, head_dim=64), rows(n_rows=n)) == rc
    for more, rc in ((dict(q_rows=(1 << 24) - 1), SMOE_OK), (dict(q_rows=1 << 24), SMOE_ERR_SHAPE),
                     (dict(n_seqs=(1 << 19) - 9), SMOE_OK), (dict(n_seqs=(1 << 19) - 8), SMOE_ERR_SHAPE),
                     (dict(k_rows=1 << 28), SMOE_OK), (dict(k_rows=1 << 28, type=smoe_amd.TYPE_F32), SMOE_ERR_SHAPE)):
        assert lib.call("attention_prompt", prompt(**more)) == rc
    for n, rc in (((1 << 19) - 1, SMOE_OK), (1 << 19, SMOE_ERR_SHAPE)):
        assert lib.call("attention_kv4", cache(), attn(n_seqs=n)) == rc


def test_lengths_of_an_append(lib):
    assert lib.call("kv4_append", cache(), rows(lens_out=DEV + 64)) == SMOE_OK
    for at in (DEV, DEV + 4, DEV - 4):
        assert lib.call("kv4_append", cache(), rows(lens_out=at)) == SMOE_ERR_ARG
    apart = dict(start=DEV, slots=DEV + 64, offsets=DEV + 128)         # 2, 2 and 3 words
    for at, rc in ((4, SMOE_ERR_ARG), (8, SMOE_OK), (60, SMOE_ERR_ARG), (68, SMOE_ERR_ARG), (72, SMOE_OK), (120, SMOE_OK),
                   (124, SMOE_ERR_ARG), (136, SMOE_ERR_ARG), (140, SMOE_OK)):
        assert lib.call("kv4_append", cache(), rows(lens_out=DEV + at, **apart)) == rc
    assert lib.call("kv4_read", cache(), rows(lens_out=DEV + 64)) == SMOE_ERR_ARG


@pytest.mark.parametrize("more,rc", [
    ({}, SMOE_OK), (dict(slots=None), SMOE_OK), (dict(max_len=0), SMOE_OK), (dict(q=None), SMOE_ERR_ARG),
    (dict(out=None), SMOE_ERR_ARG), (dict(lens=None), SMOE_ERR_ARG), (dict(n_seqs=0), SMOE_ERR_ARG),
    (dict(type=9), SMOE_ERR_ARG), (dict(scale=0.0), SMOE_ERR_ARG), (dict(num_heads=31), SMOE_ERR_SHAPE),
    (dict(num_heads=0), SMOE_ERR_SHAPE), (dict(q=DEV + 4), SMOE_ERR_SHAPE), (dict(q_stride=4094), SMOE_ERR_SHAPE),
    (dict(out_stride=4098), SMOE_ERR_SHAPE), (dict(n_seqs=1 << 27), SMOE_ERR_SHAPE),
])
def test_cache_attention(lib, more, rc):
    assert lib.call("attention_kv4", cache(), attn(**more)) == rc


def test_null_arguments(lib):
    L = lib.lib
    assert L.smoe_hip_qk_norm_rope(None, C.byref(qk())) == SMOE_ERR_ARG
    assert L.smoe_hip_attention_prompt(None, C.byref(prompt())) == SMOE_ERR_ARG
    assert L.smoe_hip_kv4_append(None, C.byref(cache()), C.byref(rows())) == SMOE_ERR_ARG
    assert L.smoe_hip_kv4_read(None, C.byref(cache()), C.byref(rows())) == SMOE_ERR_ARG
    assert L.smoe_hip_attention_kv4(None, C.byref(cache()), C.byref(attn())) == SMOE_ERR_ARG
    assert lib.call("qk_norm_rope", None) == SMOE_ERR_ARG
    assert lib.call("attention_prompt", None) == SMOE_ERR_ARG
    assert lib.call("kv4_append", None, rows()) == SMOE_ERR_ARG
    assert lib.call("kv4_read", cache(), None) == SMOE_ERR_ARG
    assert lib.call("attention_kv4", None, attn()) == SMOE_ERR_ARG
    assert lib.call("attention_kv4", cache(), None) == SMOE_ERR_ARG


def test_calls_without_rows_do_nothing(lib):
    n = lib.booked()
    L = lib.lib
    assert L.smoe_hip_qk_norm_rope(lib.ctx, C.byref(qk(n_rows=0))) == SMOE_OK
    assert L.smoe_hip_attention_prompt(lib.ctx, C.byref(prompt(q_rows=0, q=None, out=None))) == SMOE_OK
    assert L.smoe_hip_kv4_append(lib.ctx, C.byref(cache()), C.byref(rows(n_rows=0))) == SMOE_OK
    assert L.smoe_hip_kv4_read(lib.ctx, C.byref(cache()), C.byref(rows(n_rows=0))) == SMOE_OK
    assert lib.booked() == n
    # (the lengths are still wanted)
    assert lib.call("kv4_append", cache(), rows(n_rows=0, lens_out=DEV + 64)) == SMOE_OK


def test_scratch_grows_outside_capture_only(lib):
    long = dict(k_rows=9000, max_k=9000)
    lib.lib.fake_capturing(1)
    assert lib.call("attention_prompt", prompt()) == SMOE_OK              # one part: no scratch
    assert lib.call("attention_prompt", prompt(**long)) == SMOE_ERR_CAPTURE
    lib.lib.fake_capturing(0)
    assert lib.call("attention_prompt", prompt(**long)) == SMOE_OK
    held = lib.booked("part")
    lib.lib.fake_capturing(1)
    assert lib.call("attention_prompt", prompt(**long)) == SMOE_OK        # a graph may hold it now
    assert lib.booked("part") == held
    assert lib.call("attention_kv4", cache(capacity=9000), attn(max_len=9000, n_seqs=900)) == SMOE_ERR_CAPTURE
    lib.lib.fake_capturing(0)
    assert lib.call("attention_kv4", cache(capacity=9000), attn(max_len=9000, n_seqs=900)) == SMOE_OK
    assert lib.booked("part") != held and lib.lib.fake_is_live(held)


def test_scratch_that_cannot_be_had(lib):
    small = dict(max_len=600)
    assert lib.call("attention_kv4", cache(capacity=9000), attn(**small)) == SMOE_OK
    held = lib.booked("part")
    lib.lib.fake_budget(0)
    assert lib.call("attention_kv4", cache(capacity=9000), attn(max_len=9000, n_seqs=900)) == SMOE_ERR_HIP
    lib.lib.fake_budget(C.c_size_t(-1).value)
    assert lib.call("attention_kv4", cache(capacity=9000), attn(**small)) == SMOE_OK
    assert lib.booked("part") == held                                     # what was there still serves


def test_kernels_are_timed(lib):
    assert lib.lib.smoe_hip_profile_enable(lib.ctx, 1) == SMOE_OK
    assert lib.call("qk_norm_rope", qk()) == SMOE_OK
    assert lib.call("attention_prompt", prompt(k_rows=9000, max_k=9000)) == SMOE_OK
    assert lib.call("kv4_append", cache(), rows()) == SMOE_OK
    assert lib.call("kv4_read", cache(), rows()) == SMOE_OK
    assert lib.call("attention_kv4", cache(), attn()) == SMOE_OK
    for kind, n in ((smoe_amd.KERNEL_QK_ROWS, 1), (smoe_amd.KERNEL_ATTENTION_PROMPT, 1), (smoe_amd.KERNEL_KV4_ROWS, 2),
                    (smoe_amd.KERNEL_ATTENTION_KV4, 1)):
        got, ms = C.c_uint64(), C.c_double()
        assert lib.lib.smoe_hip_profile_read(lib.ctx, kind, C.byref(got), C.byref(ms)) == SMOE_OK
        assert got.value == n
