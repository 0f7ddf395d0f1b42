"""Element types of the operands that the Python entry points are given: an operand whose owner knows its type (a tensor, a
device array) has to have the one that the library reads.  No GPU: the tensors are stand-ins, and a refused call reaches
no entry point of the library."""
import numpy as np
import pytest

from cudanative_jl_b200 import gemm as G
from cudanative_jl_b200 import wmma
from cudanative_jl_b200.array import DevicePtr
from cudanative_jl_b200.bfloat16 import BFloat16

torch = pytest.importorskip("torch")

F16, F32 = np.float16, np.float32


class Tensor:
    """What the package asks of a tensor on the device."""

    is_cuda = True

    def __init__(self, dtype, rows=16, cols=16):
        self.dtype, self.shape = dtype, (cols, rows)

    def data_ptr(self):
        return 4096

    def stride(self, i):
        return (self.shape[1], 1)[i]


class Library:
    """Notes the entry points that are called; all of them succeed."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.startswith("__"):
            raise AttributeError(name)

        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


@pytest.fixture()
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(G._lib, "lib", lambda: lib)
    return lib


def handle():
    h = G.Handle.__new__(G.Handle)
    h._h, h.device = None, 0
    return h


def sharded():
    s = G.ShardedGemm.__new__(G.ShardedGemm)
    s._s, s.M, s.K = None, 16, 16
    return s


h16, f32, b16, u8, i32 = torch.float16, torch.float32, torch.bfloat16, torch.uint8, torch.int32

# entry point -> (call with operands by name, the types it reads)
ENTRIES = {
    "gemm": (lambda t: handle().gemm(False, False, 16, 16, 16, 1.0, t["A"], 16, t["B"], 16, 1.0, t["C"], 16, t["D"], 16), dict(A=h16, B=h16, C=f32, D=f32)),
    "gemm_gated": (lambda t: handle().gemm_gated(False, False, 16, 16, 16, 1.0, t["A"], 16, t["B"], 16, 1.0, t["C"], 16, t["D"], 16, t["flags"], 64),
                   dict(A=h16, B=h16, C=f32, D=f32, flags=i32)),
    "gemm_typed": (lambda t: handle().gemm_typed(False, False, 16, 16, 16, 1.0, t["A"], 16, t["B"], 16, 1.0, t["C"], 16, F16, t["D"], 16, F32),
                   dict(A=h16, B=h16, C=h16, D=f32)),
    "gemm_f16f32": (lambda t: G.gemm_f16f32(handle(), t["D"], t["A"], t["B"], t["C"], beta=1.0), dict(A=h16, B=h16, C=f32, D=f32)),
    "gemm_ex": (lambda t: handle().gemm_ex(False, False, 16, 16, 16, 1.0, t["A"], 16, t["B"], 16, BFloat16, 1.0, t["C"], 16, F16, t["D"], 16, BFloat16),
                dict(A=b16, B=b16, C=h16, D=b16)),
    "gemm_strided_batched": (lambda t: handle().gemm_strided_batched(False, False, 16, 16, 16, 1.0, t["A"], 16, 256, t["B"], 16, 256, F16, 1.0, t["C"], 16, 256, F32,
                                                                     t["D"], 16, 256, F16, 2), dict(A=h16, B=h16, C=f32, D=h16)),
    "gemm_grouped": (lambda t: handle().gemm_grouped(True, 16, 16, 16, 1.0, t["A"], 16, 256, t["B"], 16, BFloat16, 1.0, t["C"], 16, F32, t["D"], 16, F16,
                                                     t["offsets"], 2), dict(A=b16, B=b16, C=f32, D=h16, offsets=i32)),
    "gemm_grouped_k": (lambda t: handle().gemm_grouped_k(16, 16, 16, 1.0, t["A"], 16, t["B"], 16, F16, 1.0, t["C"], 16, 256, BFloat16, t["D"], 16, 256,
                                                         F32, t["offsets"], 2), dict(A=h16, B=h16, C=b16, D=f32, offsets=i32)),
    "mxfp4_quantize": (lambda t: handle().mxfp4_quantize(False, 32, 16, t["X"], 32, BFloat16, t["Q"], 32, t["scales"], t["offsets"], 2),
                       dict(X=b16, Q=u8, scales=u8, offsets=i32)),
    "mxfp4_dequantize": (lambda t: handle().mxfp4_dequantize(32, 16, t["Q"], 32, t["scales"], t["Y"], 32, F32, t["offsets"], 2),
                         dict(Q=u8, scales=u8, Y=f32, offsets=i32)),
    "gemm_mxfp4": (lambda t: handle().gemm_mxfp4(16, 16, 32, 1.0, t["A"], 32, t["SA"], t["B"], 32, t["SB"], 1.0, t["C"], 16, F32, t["D"], 16, BFloat16),
                   dict(A=u8, SA=u8, B=u8, SB=u8, C=f32, D=b16)),
    "gemm_mxfp4_grouped": (lambda t: handle().gemm_mxfp4_grouped(16, 16, 32, 1.0, t["A"], 32, 512, t["SA"], t["B"], 32, t["SB"], 1.0, t["C"], 16, F16, t["D"],
                                                                 16, F32, t["offsets"], 2), dict(A=u8, SA=u8, B=u8, SB=u8, C=h16, D=f32, offsets=i32)),
    "ShardedGemm.run": (lambda t: sharded().run(1.0, t["B"], 1.0, t["C"], t["D"]), dict(B=h16, C=f32, D=f32)),
}
# gemm_f16f32 takes the types of C and D from the operands; flags are any 32-bit words
FREE = {("gemm_gated", "flags"): (i32, f32), ("gemm_f16f32", "C"): (h16, f32), ("gemm_f16f32", "D"): (h16, f32)}


@pytest.mark.parametrize("entry", ENTRIES)
def test_the_right_types_reach_the_library(library, entry):
    call, types = ENTRIES[entry]
    call({k: Tensor(t) for k, t in types.items()})
    assert len(library.calls) == 1


ALL = [h16, f32, b16, u8, i32, torch.int64, torch.float64]
WRONG = [(e, o, w) for e, (_, types) in ENTRIES.items() for o, t in types.items() for w in ALL if w not in FREE.get((e, o), (t,))]


@pytest.mark.parametrize("entry,operand,wrong", WRONG, ids=str)
def test_another_type_is_refused(library, entry, operand, wrong):
    call, types = ENTRIES[entry]
    with pytest.raises(TypeError):
        call({**{k: Tensor(t) for k, t in types.items()}, operand: Tensor(wrong)})
    assert not library.calls


@pytest.mark.parametrize("entry", ENTRIES)
def test_addresses_and_typed_pointers(library, entry):
    """An address has no type; a DevicePtr has one, bfloat16 being its bit patterns."""
    call, types = ENTRIES[entry]
    stored = {h16: F16, f32: F32, b16: np.uint16, u8: np.uint8, i32: np.int32}
    call({k: DevicePtr(stored[t], 4096) if entry != "gemm_f16f32" else Tensor(t) for k, t in types.items()})
    if entry != "gemm_f16f32":
        call({k: 4096 for k in types})
    if entry in ("gemm_ex", "gemm_strided_batched"):  # a buffer of what the tags say
        call({k: DevicePtr(np.int8, 4096) for k in types})
    elif entry != "gemm_f16f32":
        with pytest.raises(TypeError):
            call({k: DevicePtr(np.int8, 4096) for k in types})


def test_offsets_of_64_bits_are_refused(library):
    """Read as 32 bits, 0, 0, n, 0 would be a legal empty group: nothing written, nothing reported."""
    for name in ("gemm_grouped", "gemm_grouped_k", "mxfp4_quantize", "mxfp4_dequantize", "gemm_mxfp4_grouped"):
        call, types = ENTRIES[name]
        with pytest.raises(TypeError, match="offsets: expected int32"):
            call({**{k: Tensor(t) for k, t in types.items()}, "offsets": DevicePtr(np.int64, 4096)})
    assert not library.calls


def test_a_c_that_is_not_read_has_any_type(library):
    handle().gemm(False, False, 16, 16, 16, 1.0, Tensor(h16), 16, Tensor(h16), 16, 0.0, Tensor(h16), 16, Tensor(f32), 16)
    assert len(library.calls) == 1


def test_the_16x16x16_unit_refuses_other_types(library):
    for c, d in ((Tensor(u8), Tensor(f32)), (Tensor(f32), Tensor(i32)), (None, Tensor(b16))):
        with pytest.raises(ValueError, match="Invalid element type"):
            wmma.wmma_16x16x16(Tensor(h16), Tensor(h16), c, d)
    with pytest.raises(ValueError, match="Invalid element type"):
        wmma.wmma_16x16x16(Tensor(b16), Tensor(h16), None, Tensor(f32))
    assert not library.calls
