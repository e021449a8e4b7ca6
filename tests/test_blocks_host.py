"""CPU tests of the token-block operators' argument checks (sga_amd.blocks and the C entry points): a call that cannot be carried
out is refused before anything is launched."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import torch

import sga_amd  # noqa: F401
from sga_amd import _lib, blocks

P = 1 << 20      # an address that no check reads


def linear(**kw):
    a = _lib.SgaLinear(rows=4, in_features=8, out_features=16, dtype=1, act=0, x=P, ld_x=8, w=P, ld_w=8, out=P, ld_out=16, ld_residual=16,
                       g_out=P, ld_g_out=16, g_x=P, g_w=P, g_bias=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD, UNSUPPORTED, NOMEM = -1, -3, -6


@pytest.mark.parametrize("change,status", [
    ({"rows": -1}, BAD), ({"in_features": 0}, BAD), ({"out_features": 0}, BAD), ({"dtype": 3}, BAD), ({"dtype": -1}, BAD), ({"act": 5}, BAD),
    ({"ld_x": 7}, BAD), ({"ld_x": -8}, BAD), ({"ld_w": 4}, BAD), ({"x": P + 1}, BAD), ({"w": P + 1}, BAD),
    ({"in_features": (1 << 20) + 1, "ld_x": 1 << 21, "ld_w": 1 << 21}, UNSUPPORTED), ({"rows": 1 << 31}, UNSUPPORTED),
    ({"dropout": _lib.SgaDropout(-0.1, 0, 0, None)}, BAD), ({"dropout": _lib.SgaDropout(1.1, 0, 0, None)}, BAD),
    ({"dropout": _lib.SgaDropout(float("nan"), 0, 0, None)}, BAD), ({"dropout": _lib.SgaDropout(0.5, 0, 0, P + 4)}, BAD)])
def test_linear_refuses(change, status):
    lib = _lib.load_library()
    n = C.c_int64(0)
    for backward in (0, 1):
        assert lib.sga_op_linear_workspace(C.byref(linear(**change)), backward, C.byref(n)) == status
    assert lib.sga_op_linear_fwd(C.byref(linear(**change)), None, 0, None) == status
    assert lib.sga_op_linear_bwd(C.byref(linear(**change)), None, 0, None) == status


@pytest.mark.parametrize("change", [{"x": None}, {"w": None}, {"out": None}, {"ld_out": 15}, {"ld_out": 0}, {"residual": P, "ld_residual": 3},
                                    {"bias": P + 1}, {"residual": P + 1}, {"out": P + 1}])
def test_linear_forward_refuses(change):
    assert _lib.load_library().sga_op_linear_fwd(C.byref(linear(**change)), None, 0, None) == BAD


@pytest.mark.parametrize("change", [{"g_out": None}, {"act": 2}, {"x": None}, {"w": None}, {"ld_g_out": 15}, {"g_x": P + 1}, {"g_bias": P + 1}])
def test_linear_backward_refuses(change):
    assert _lib.load_library().sga_op_linear_bwd(C.byref(linear(**change)), P, 1 << 30, None) == BAD


def test_linear_refuses_null_and_small_workspaces():
    lib = _lib.load_library()
    n = C.c_int64(0)
    assert lib.sga_op_linear_workspace(None, 0, C.byref(n)) == BAD
    assert lib.sga_op_linear_workspace(C.byref(linear()), 0, None) == BAD
    assert lib.sga_op_linear_fwd(None, None, 0, None) == BAD
    a = linear(act=2, pre=P)
    assert lib.sga_op_linear_workspace(C.byref(a), 1, C.byref(n)) == 0 and n.value > 0
    assert lib.sga_op_linear_bwd(C.byref(a), P, n.value - 1, None) == NOMEM
    assert lib.sga_op_linear_bwd(C.byref(a), None, n.value, None) == NOMEM
    assert lib.sga_op_linear_bwd(C.byref(a), P + 8, n.value, None) == NOMEM


def norm(**kw):
    a = _lib.SgaLayerNorm(rows=4, cols=8, dtype=1, param_dtype=0, eps=1e-5, x=P, ld_x=8, y=P, mean=P, rstd=P, g_y=P, ld_g_y=8, g_x=P, g_w=P, g_b=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    ({"rows": -1}, BAD), ({"cols": 0}, BAD), ({"dtype": 3}, BAD), ({"param_dtype": 2}, BAD), ({"ld_x": 7}, BAD), ({"x": P + 1}, BAD), ({"w": P + 2}, BAD),
    ({"x": None}, BAD), ({"mean": P + 2}, BAD), ({"cols": (1 << 20) + 1, "ld_x": 1 << 21}, UNSUPPORTED), ({"rows": 1 << 31}, UNSUPPORTED)])
def test_layer_norm_refuses(change, status):
    lib = _lib.load_library()
    n = C.c_int64(0)
    for backward in (0, 1):
        assert lib.sga_op_layer_norm_workspace(C.byref(norm(**change)), backward, C.byref(n)) == status
    assert lib.sga_op_layer_norm_fwd(C.byref(norm(**change)), None) == status
    assert lib.sga_op_layer_norm_bwd(C.byref(norm(**change)), P, 1 << 30, None) == status


def test_layer_norm_refuses_by_direction():
    lib = _lib.load_library()
    n = C.c_int64(0)
    for change in ({"eps": -1.0}, {"eps": float("nan")}, {"y": None}, {"y": P + 1}):
        assert lib.sga_op_layer_norm_fwd(C.byref(norm(**change)), None) == BAD
    for change in ({"g_y": None}, {"mean": None}, {"rstd": None}, {"ld_g_y": 3}, {"g_add": P, "ld_g_add": 3}, {"g_x": P + 1}, {"g_w": P + 2}):
        assert lib.sga_op_layer_norm_bwd(C.byref(norm(**change)), P, 1 << 30, None) == BAD
    assert lib.sga_op_layer_norm_workspace(C.byref(norm()), 1, C.byref(n)) == 0 and n.value > 0
    assert lib.sga_op_layer_norm_bwd(C.byref(norm()), P, n.value - 1, None) == NOMEM
    assert lib.sga_op_layer_norm_bwd(C.byref(norm()), None, 0, None) == NOMEM


def test_dropout_refuses():
    lib = _lib.load_library()

    def call(x=P, ld_x=8, res=None, ld_res=8, y=P, rows=4, cols=8, dtype=1, p=0.5, state=None, drop=True):
        d = _lib.SgaDropout(p, 1, 0, state)
        return lib.sga_op_dropout(x, ld_x, res, ld_res, y, rows, cols, dtype, C.byref(d) if drop else None, None)

    for kw in ({"x": None}, {"y": None}, {"ld_x": 7}, {"res": P, "ld_res": 7}, {"rows": -1}, {"cols": 0}, {"dtype": 3}, {"p": -1.0}, {"p": 2.0},
               {"state": P + 1}, {"drop": False}, {"x": P + 1}, {"y": P + 1}, {"res": P + 1}):
        assert call(**kw) == BAD, kw
    assert call(rows=1 << 31) == UNSUPPORTED
    assert call(x=None, y=None, rows=0) == 0


def test_python_refuses_before_it_asks_for_a_gpu():
    x, w = torch.ones(4, 8), torch.ones(16, 8)
    with pytest.raises(ValueError, match="on the GPU"):
        blocks.linear(x, w)
    with pytest.raises(TypeError):
        blocks.linear(x.double(), w)
    with pytest.raises(TypeError):
        blocks.linear([1.0], w)
    with pytest.raises(ValueError, match="adjacent"):
        blocks.layer_norm(torch.ones(8, 4).t())
    with pytest.raises(ValueError, match="common stride"):
        blocks.layer_norm(torch.ones(4, 6, 8)[:, ::2][:3, :2])
    with pytest.raises(ValueError, match="overlap"):
        blocks.layer_norm(torch.ones(100).as_strided((4, 8), (3, 1)))
    with pytest.raises(ValueError, match="at least one feature"):
        blocks.layer_norm(torch.ones(4, 0))
    with pytest.raises(ValueError, match="at least one feature"):
        blocks.dropout(torch.tensor(1.0), 0.5, 1)
    with pytest.raises(ValueError, match="act"):
        blocks._act("tanh")
    for bad in ((-0.5, 1, 0), (1.5, 1, 0), (float("nan"), 1, 0), (0.5, 1), (0.5, torch.zeros(2))):
        with pytest.raises(ValueError):
            blocks._drop(bad, torch.device("cpu"))
    assert blocks._drop((0.5, -1, 1 << 65), torch.device("cpu")) == (0.5, (1 << 64) - 1, 0, 0)


def test_packed_arguments_are_the_structures():
    """blocks passes the structures of include/sga_hip.h as packed bytes: the same bytes as the ctypes structures hold."""
    drop = (0.25, 3, 4, 5 << 12)
    v = [7, 8, 9, 1, 2] + [P + 16 * i for i in range(15)]
    a = _lib.SgaLinear(*v, _lib.SgaDropout(*drop))
    assert blocks._LINEAR(*v, *drop) == bytes(a)
    v = [7, 8, 1, 0, 0.5] + [P + 16 * i for i in range(14)]
    assert blocks._NORM(*v) == bytes(_lib.SgaLayerNorm(*v))
    assert blocks._DROPOUT(*drop) == bytes(_lib.SgaDropout(*drop))


def test_row_layouts():
    """Rows of wider buffers, repeated rows and batches collapse to (rows, features, row stride); checked up to the device."""
    def layout(t):
        try:
            blocks._rows(t, "t")
        except ValueError as e:
            return "GPU" in str(e)      # everything but the device is in order
        raise AssertionError
    base = torch.ones(6, 40)
    for t in (base, base[:, 3:20], base[::2], base[:1].expand(5, 40), base.view(2, 3, 40), base.view(2, 3, 40)[:, :, :8], torch.ones(8), base[:, :1],
              torch.ones(0, 8), base[2:3, 1:9], base.view(2, 3, 40)[:1, ::2]):
        assert layout(t), t.shape
    for t in (base.t(), base.view(2, 3, 40)[:, :2], base.expand(3, 6, 40)):
        assert not layout(t), t.shape


def scalar_registers(operand):
    m = re.fullmatch(r"s(\d+)|s\[(\d+):(\d+)\]", operand.split(" ")[0])
    if not m:
        return ()
    return (int(m.group(1)),) if m.group(1) else range(int(m.group(2)), int(m.group(3)) + 1)


def short_waits(asm):
    """-> (fetches into LDS, [(kernel, wait states, writer, fetch)] with fewer than 5 wait states between a vector instruction that
    writes a scalar register and a vector memory instruction that uses it; the same for m0 and a fetch into LDS: fewer than 1).
    Straight lines: every instruction is one wait state, s_nop n is n + 1."""
    kernel, at, wrote, m0, fetches, short = None, 0, {}, -9, 0, []
    for line in asm.splitlines():
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            kernel, wrote, m0 = m.group(1), {}, -9
            continue
        text = line.split("//")[0].strip()
        if not line.startswith("\t") or not text:
            continue
        op, _, rest = text.partition(" ")
        args = [a.strip() for a in rest.split(",")]
        if op.startswith(("buffer_", "global_", "flat_", "scratch_")):
            used = [r for a in args for r in scalar_registers(a)]
            short += [(kernel, at - wrote[r][0] - 1, wrote[r][1], text) for r in used if r in wrote and at - wrote[r][0] - 1 < 5]
            if text.endswith(" lds"):
                fetches += 1
                if at - m0 - 1 < 1:
                    short.append((kernel, 0, "m0", text))
        elif op.startswith("v_"):
            carries = op.startswith(("v_cmp", "v_add_co", "v_sub_co", "v_subrev_co", "v_addc", "v_subb", "v_mad_u64", "v_mad_i64", "v_div_scale"))
            for a in args[:2 if carries else 1]:
                wrote.update((r, (at, text)) for r in scalar_registers(a))
        elif op.startswith("s_"):
            for r in scalar_registers(args[0]):
                wrote.pop(r, None)
            if args[0] == "m0":
                m0 = at
        at += int(args[0], 0) + 1 if op == "s_nop" else 1
    return fetches, short


def test_wait_states_are_counted():
    """The counter itself, on lines with and without the waits."""
    def lines(*ops):
        return "0000 <k>:\n" + "\n".join("\t%s // x" % o for o in ops)
    fetch = "buffer_load_dwordx4 v9, s[4:7], 0 offen lds"
    start = ["v_readfirstlane_b32 s4, v1", "s_add_u32 s8, s8, s9", "s_mov_b32 m0, s10"]
    assert short_waits(lines(*start, "s_nop 0", fetch))[1][0][1] == 3
    assert short_waits(lines(*start, "s_nop 1", fetch))[1][0][1] == 4
    assert short_waits(lines(*start, "s_nop 2", fetch)) == (1, [])
    assert short_waits(lines("s_mov_b32 m0, s10", fetch))[1][0][2] == "m0"
    assert short_waits(lines("v_readlane_b32 s4, v1, 3", "s_mov_b32 s4, s5", fetch.replace(" lds", ""))) == (0, [])      # written again by a scalar instruction
    assert short_waits(lines("v_cmp_lt_u32_e64 s[6:7], v1, v2", fetch.replace(" lds", "")))[1]


def test_fetches_into_lds_wait_for_their_scalar_registers(tmp_path):
    """The matrix product's fetches are written by hand, where the compiler keeps no distances: every one of the built library has them."""
    llvm = "/opt/rocm/lib/llvm/bin"
    bundler, objdump = os.path.join(llvm, "clang-offload-bundler"), os.path.join(llvm, "llvm-objdump")
    if not (os.path.exists(bundler) and os.path.exists(objdump) and shutil.which("objcopy")):
        pytest.skip("no ROCm LLVM tools here")
    fat = tmp_path / "fat.bin"
    subprocess.run(["objcopy", "-O", "binary", "--only-section=.hip_fatbin", _lib.LIB_PATH, str(fat)], check=True)
    data, total, short = fat.read_bytes(), 0, []
    starts = [m.start() for m in re.finditer(re.escape(b"__CLANG_OFFLOAD_BUNDLE__"), data)] + [len(data)]
    for b, e in zip(starts, starts[1:]):
        one, co = tmp_path / "one.bin", tmp_path / "one.co"
        one.write_bytes(data[b:e])
        subprocess.run([bundler, "--unbundle", "--type=o", "--input=%s" % one, "--output=%s" % co, "--targets=hipv4-amdgcn-amd-amdhsa--gfx950"],
                       check=True, capture_output=True)
        asm = subprocess.run([objdump, "-d", str(co)], check=True, capture_output=True, text=True).stdout
        n, s = short_waits(asm)
        total += n
        short += s
    assert total > 500 and not short, (total, len(short), short[:4])


def test_parameter_types_of_a_norm():
    """weight and bias have x's type or float32, whichever of them is given; anything else is a TypeError."""
    for x in (torch.float32, torch.bfloat16, torch.float16):
        assert blocks._param_type(None, None, x) == x
        for t in (x, torch.float32):
            p = torch.ones(4, dtype=t)
            assert blocks._param_type(p, None, x) == blocks._param_type(None, p, x) == blocks._param_type(p, p, x) == t
        for t in {torch.float64, torch.int32, torch.bool, torch.float16, torch.bfloat16} - {x}:
            p = torch.ones(4).to(t)
            for args in ((p, None), (None, p), (p, torch.ones(4))):
                with pytest.raises(TypeError):
                    blocks._param_type(*args, x)
        for args in (([1.0] * 4, None), (None, [1.0] * 4), (None, 1.0)):
            with pytest.raises(TypeError):
                blocks._param_type(*args, x)


def test_linear_row_limit():
    """More rows than the tiles of one launch can cover are refused, up to there they are not."""
    lib = _lib.load_library()
    n = C.c_int64(0)
    most = (1 << 31) - 256
    for backward in (0, 1):
        for features in (1, 8):
            a = dict(in_features=features, out_features=features)
            assert lib.sga_op_linear_workspace(C.byref(linear(rows=most, **a)), backward, C.byref(n)) == 0
            assert lib.sga_op_linear_workspace(C.byref(linear(rows=most + 1, **a)), backward, C.byref(n)) == UNSUPPORTED
    assert lib.sga_op_linear_fwd(C.byref(linear(rows=most + 1)), None, 0, None) == UNSUPPORTED
    assert lib.sga_op_linear_bwd(C.byref(linear(rows=most + 1)), P, 1 << 62, None) == UNSUPPORTED
