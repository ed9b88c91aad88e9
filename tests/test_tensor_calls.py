"""The host module that passes tensors to the library's entry points: what it takes for which argument, that it refuses what the
checks in Python refuse, and that the calls it makes are theirs."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tinyserve_b200.kernels import build, ops

CALLS = [v for v in vars(ops).values() if isinstance(v, ops._TensorCall)]


@pytest.fixture(scope="module")
def module():
    m = build.calls()
    if m is None:
        pytest.skip("no host module (built without Python's or PyTorch's headers)")
    return m


def test_patterns_fit_the_entry_points(module) -> None:
    lib = build.library()
    lib.ts_list_function.argtypes, lib.ts_list_function.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_void_p
    assert len(CALLS) == 7
    for c in CALLS:
        kinds = ctypes.create_string_buffer(65)
        at = lib.ts_list_function(c.name.encode(), ctypes.addressof(kinds))
        assert at and len(kinds.value) == len(c.pattern) == len(ops._SIGNATURES[c.name])
        assert sum(p in "d8fiDFI" for p in c.pattern) == len(c.names)
        module.Call(at, kinds.value.decode(), c.pattern)
        with pytest.raises(ValueError):
            module.Call(at, kinds.value.decode(), c.pattern[:-1])
        with pytest.raises(ValueError):
            module.Call(at, kinds.value.decode(), "n" * len(c.pattern))
    assert lib.ts_list_function(b"ts_no_such_function", ctypes.addressof(kinds)) is None


def test_without_a_compiler_or_the_cuda_headers_calls_go_through_ctypes(monkeypatch, tmp_path) -> None:
    """A machine that has the built library and no toolkit, or no g++: no module, and no error."""
    def none() -> str:
        raise build.KernelBuildError("nvcc not found")

    with monkeypatch.context() as m:
        m.setattr(build, "find_nvcc", none)
        assert build.build_calls(tmp_path) is None
        m.setattr(build, "_calls", [])
        m.setattr(build, "build_dir", lambda: tmp_path)
        assert build.calls() is None
    monkeypatch.setenv("PATH", str(tmp_path))
    assert build.build_calls(tmp_path) is None
    assert not list(tmp_path.iterdir())


SEEN: list[int] = []
WORDS = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(ctypes.c_uint64))


@WORDS
def take(words):
    SEEN[:] = [words[i] for i in range(6)]
    return 7


def test_words_and_refusals(module) -> None:
    """On the CPU no tensor is taken (they have to lie on the device); numbers, addresses and None become their words."""
    at = ctypes.cast(take, ctypes.c_void_p).value
    call = module.Call(at, "pilfpp", "Dnnxpp")
    assert call(None, -3, 1 << 40, 0.5, 2 ** 63 + 5, 0) == 7
    assert SEEN == [0, 2 ** 64 - 3, 1 << 40, int.from_bytes(bytes(memoryview(ctypes.c_float(0.5))), "little"), 2 ** 63 + 5, 0]
    assert call(None, 2 ** 31, 0, 0.0, 0, 0) == module.NOT_TAKEN               # no 32-bit integer
    assert call(torch.zeros(3), 1, 0, 0.0, 0, 0) == module.NOT_TAKEN           # not on the device
    assert call(7, 1, 0, 0.0, 0, 0) == module.NOT_TAKEN                        # no tensor
    with pytest.raises(TypeError):
        call(None, 1, 0, 0.0, 0)
    with pytest.raises(TypeError):
        call(None, "1", 0, 0.0, 0, 0)
    with pytest.raises(TypeError):
        call(None, 1, 0, 0.0, 0, p=0)
    with pytest.raises(OverflowError):
        call(None, 1 << 70, 0, 0.0, 0, 0)


def test_sizes_beyond_32_bits_are_refused(monkeypatch) -> None:
    """Where the host module does not take a call it is made through ctypes, which would cut such a size off without a word."""
    made = []
    monkeypatch.setattr(ops, "_dev", lambda t, name, dtype=None: 16)
    monkeypatch.setattr(ops, "_fn", lambda name: lambda *words: made.append(words) or 0)
    x, codes, scales = torch.zeros(1), torch.zeros(1, dtype=torch.int8), torch.zeros(1)
    call = ops._TensorCall("ts_act_mul_int8", "act_mul_int8", "d8fnnnn=p", "x out scales")
    for sizes in ((2 ** 31, 64, 64, 3), (5, 64, 2 ** 32 + 64, 3), (-2 ** 31 - 1, 64, 64, 3)):
        with pytest.raises(ops.KernelError, match="act_mul_int8: .* 32 bits"):
            call._by_ctypes((x, codes, scales, *sizes, 0))
    assert not made
    call._by_ctypes((x, codes, scales, 2 ** 31 - 1, 64, 64, 3, 2 ** 48))       # an address may be as large as it is
    assert len(made) == 1 and made[0][3] == 2 ** 31 - 1 and made[0][-1] == 2 ** 48


@pytest.mark.gpu
def test_only_what_fits_is_taken(module) -> None:
    at = ctypes.cast(take, ctypes.c_void_p).value
    call = module.Call(at, "ppppip", "d8fI=D")
    z = dict(device="cuda")
    b, i8, f, i32 = torch.zeros(4, 8, dtype=torch.bfloat16, **z), torch.zeros(4, dtype=torch.int8, **z), torch.zeros(4, **z), torch.zeros(4, dtype=torch.int32, **z)
    assert call(b, i8, f, i32, b) == 7
    assert SEEN == [b.data_ptr(), i8.data_ptr(), f.data_ptr(), i32.data_ptr(), 1, b.data_ptr()]
    assert call(f, i8, f, None, None) == 7 and SEEN[3:] == [0, 0, 0]
    assert call(b[1:], i8, f, None, None) == 7 and SEEN[0] == b.data_ptr() + 16
    for wrong in ((b, i8, f, None, f), (b.half(), i8, f, None, None), (b.t(), i8, f, None, None), (b, f, f, None, None), (b, i8.to(torch.uint8), f, None, None),
                  (b, i8, f.double(), None, None), (b, i8, f, i32.long(), None), (b.cpu(), i8, f, None, None), (None, i8, f, None, None), (b, i8, None, None, None)):
        assert call(*wrong) == module.NOT_TAKEN


@pytest.mark.gpu
def test_the_same_calls_through_ctypes(module, monkeypatch) -> None:
    """A call made by the host module and one made through ctypes: the same results, counts and errors."""
    x = torch.randn(5, 64, device="cuda")
    outs = []
    for through in (True, False):
        codes, scales = torch.empty(5, 64, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
        call = ops._TensorCall("ts_act_mul_int8", "act_mul_int8", "d8fnnnn=p", "x out scales")
        call._bind()
        if not through:
            call._fast = None
        before = ops.launch_count
        call(x, codes, scales, 5, 64, 64, 3, ops._stream())
        assert ops.launch_count == before + 1
        outs.append((codes, scales))
        for args, match in (((x.half(), codes, scales), "dtype"), ((x, codes.int(), scales), "out must be torch.int8"), ((x, codes, scales.cpu()), "scales must be a CUDA"),
                            ((x.t(), codes, scales), "x must be contiguous")):
            with pytest.raises(ops.KernelError, match=match):
                call(*args, 5, 64, 64, 3, ops._stream())
        with pytest.raises(ops.KernelError, match="bad argument"):
            call(x, codes, scales, 5, 64, 64, 9, ops._stream())
    assert all(torch.equal(a, b) for a, b in zip(*outs))
