"""The C entry points of the windowed serving step (include/kushkash_amd_window.h, include/kushkash_amd_step.h) on the CPU, with no
GPU call: their argument lists against the Python binding's, their refusals, the windowed decode's assembly by the rules
that the plain decode's keeps, and the native host side (csrc/kush_stepcall.cpp) around entry points that only count."""
import ctypes
import re
import shutil
import subprocess
import sys
import types
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

import kushkash_amd
import test_isa as isa
from kushkash_amd import _lib

INCLUDE = Path(__file__).resolve().parent.parent / "include"
KINDS = {"int": ctypes.c_int32, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float,
         "double": ctypes.c_double}


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB.exists():
        kushkash_amd.build()
    return _lib.lib()


def declared(header: str) -> dict[str, tuple[str, list[str]]]:
    """name -> (result type, parameter declarations) of every function of a header."""
    text = re.sub(r"/\*.*?\*/", "", (INCLUDE / header).read_text(), flags=re.S)
    return {m.group(2): (m.group(1), [" ".join(p.split()) for p in m.group(3).split(",")])
            for m in re.finditer(r"\b(int|int64_t)\s+(kush_\w+)\s*\(([^)]*)\)\s*;", text)}


@pytest.mark.parametrize("header, signatures", [("kushkash_amd_window.h", _lib.WINDOW_SIGNATURES),
                                                ("kushkash_amd_step.h", _lib.STEP_SIGNATURES)])
def test_library_exports_the_headers(lib, header, signatures):
    fns = declared(header)
    assert set(fns) == set(signatures)
    for name, (result, params) in fns.items():
        want = [ctypes.c_void_p if "*" in p else KINDS[p.split()[0]] for p in params]
        assert signatures[name] == want == getattr(lib, name).argtypes, name
        assert getattr(lib, name).restype is KINDS[result]


def test_the_windowed_calls_extend_the_plain_ones():
    """kush_window_decode is kush_append_decode's list, and kush_window_attend kush_attend's without causal, with window and
    sinks (and the row tiles) behind them."""
    names = lambda ps: [re.sub(r"\W", "", p.split()[-1]) for p in ps]  # noqa: E731
    text = re.sub(r"/\*.*?\*/", "", (INCLUDE / "kushkash_amd.h").read_text(), flags=re.S)
    plain = re.search(r"int kush_append_decode\(([^)]*)\)", text).group(1).split(",")
    window = declared("kushkash_amd_window.h")
    assert names(window["kush_window_decode"][1]) == names(plain) + ["window", "sinks"]
    text = re.sub(r"/\*.*?\*/", "", (INCLUDE / "kushkash_amd_attend.h").read_text(), flags=re.S)
    plain = [n for n in names(re.search(r"int kush_attend\(([^)]*)\)", text).group(1).split(",")) if n != "causal"]
    assert names(window["kush_window_attend"][1]) == plain + ["window", "sinks", "row_tiles"]


def refused(lib, name, args, code, msg):
    assert getattr(lib, name)(*args) == code, (name, lib.kush_last_error())
    assert msg in lib.kush_last_error().decode()


def test_window_decode_refuses_bad_arguments(lib):
    base = dict(head_dim=128, bits=4, group=7, dtype=2, q=None, out=None, cache=None, bs=0, hs=0, tail_k=None, tail_idx=None,
                bt=None, seq_lens=None, bt_stride=0, hkv=4, scale=1.0, n_splits=1, part_ml=None, part_o=None, n_seqs=1,
                stream=None, k=None, v=None, ks=0, vs=0, bt_cols=0, sync=None, waves=0, seq_order=None, rot=0, window=5, sinks=0)
    for kw, code, msg in [(dict(window=0), -2, "bad window"), (dict(window=-3), -2, "bad window"), (dict(sinks=-1), -2, "bad window"),
                          (dict(k=16), -2, "go together"), (dict(v=16), -2, "go together"), (dict(k=16, v=16, group=17), -2, "group 17 > 16"),
                          (dict(k=8, v=16), -2, "aligned"), (dict(k=16, v=16, vs=3), -2, "aligned"),
                          (dict(head_dim=96), -1, "unsupported head_dim"), (dict(bits=3), -1, "unsupported bits"),
                          (dict(dtype=7), -1, "unsupported dtype"), (dict(n_seqs=-1), -2, "bad n_seqs"), (dict(n_splits=4), -2, "partial buffers"),
                          (dict(bs=8), -2, "16-byte aligned"), (dict(waves=3), -2, "waves"), (dict(rot=2), -2, "rot")]:
        refused(lib, "kush_window_decode", list({**base, **kw}.values()), code, msg)
    assert lib.kush_window_decode(*{**base, "n_seqs": 0}.values()) == 0


def test_window_attend_refuses_bad_arguments(lib):
    st = (ctypes.c_int64 * 15)(*[128 * 4, 128, 128] * 4)
    base = dict(head_dim=128, dtype=2, q=None, k=None, v=None, out=None, lse=None, strides=st, cu_q=None, cu_k=None, n_q=4, n_k=9,
                total_q=4, n_seqs=1, hkv=1, group=1, scale=1.0, out_f32=0, waves=4, chunk=0, part_o=None, part_ml=None, stream=None,
                window=3, sinks=0, row_tiles=0)
    for kw, code, msg in [(dict(window=0), -2, "bad window"), (dict(sinks=-1), -2, "bad window"), (dict(row_tiles=-1), -2, "bad window"),
                          (dict(row_tiles=3), -2, "row_tiles"), (dict(n_k=3), -2, "n_k >= n_q"), (dict(scale=0.0), -2, "scale"),
                          (dict(dtype=0), -1, "dtype"), (dict(chunk=1, n_k=200), -2, "partial buffers"), (dict(q=8), -2, "aligned"),
                          (dict(strides=(ctypes.c_int64 * 15)(*[64] * 15)), -2, "row strides"), (dict(head_dim=96), -1, "head_dim"),
                          (dict(cu_q=16), -2, "bad n_seqs"), (dict(group=0), -2, "bad n_seqs")]:
        refused(lib, "kush_window_attend", list({**base, **kw}.values()), code, msg)
    assert lib.kush_window_attend(*{**base, "n_seqs": 0}.values()) == 0


def test_step_entry_points_refuse_bad_arguments(lib):
    table = [None, 0, 5, 64, None, 0, None, 0, 2, 2, None, 2, None, None, None]
    for at, x in ((2, -1), (3, -1), (8, -1), (9, -1), (9, 65535 * 256 + 1), (11, 1)):
        refused(lib, "kush_block_table", table[:at] + [x] + table[at + 1:], -2, "kush_block_table: bad")
    assert lib.kush_block_table(*table[:8], 0, *table[9:]) == 0
    maps = [None, None, None, None, 0, 0, 2, 0, 0, 1, 1, 1, 1] + [None] * 12
    for at, x in ((6, -1), (6, 65537), (7, -1), (8, -1), (9, -1), (10, 1 << 31), (11, -1), (12, 1 << 31)):
        refused(lib, "kush_step_maps", maps[:at] + [x] + maps[at + 1:], -2, "kush_step_maps: bad")
    assert lib.kush_step_maps(*maps[:6], 0, *maps[7:]) == 0
    one = [0, None, 100, 2, 100, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None, 4096, lib.kush_sample_scratch(2, 100), None]
    for at, x, code, msg in ((0, 3, -1, "dtype"), (0, -1, -1, "dtype"), (2, -1, -2, "row_stride"), (3, -1, -2, "bad rows"),
                             (4, 0, -2, "vocab"), (4, (1 << 24) + 1, -2, "vocab"), (15, None, -2, "scratch"), (15, 4104, -2, "scratch"),
                             (16, lib.kush_sample_scratch(2, 100) - 1, -2, "scratch")):
        refused(lib, "kush_sample", one[:at] + [x] + one[at + 1:], code, msg)
    assert lib.kush_sample(*one[:3], 0, *one[4:]) == 0
    for rows, vocab in ((-1, 5), (2, 0), (2, (1 << 24) + 1)):
        assert lib.kush_sample_scratch(rows, vocab) == 0
    # one launch's rows at most, whatever the batch; within a megabyte a row at the largest vocabulary
    assert lib.kush_sample_scratch(1 << 20, 1000) == lib.kush_sample_scratch(1024, 1000)
    assert 0 < lib.kush_sample_scratch(1, 1 << 24) < 1 << 20


# ------------------------------------------------------------------ assembly
@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not available")
    from kushkash_amd.build import DECODE_INST, FLAGS
    tmp = tmp_path_factory.mktemp("isa")
    src = isa.SRC.with_name("kush_window_inst.hip")

    def compile_one(i_defs):
        out = tmp / f"w{i_defs[0]}.s"
        subprocess.run([hipcc, *(f for f in FLAGS if f not in ("-shared", "-fPIC")), *(f"-D{k}={v}" for k, v in i_defs[1].items()),
                        f"-I{INCLUDE}", "-S", "--cuda-device-only", str(src), "-o", str(out)], check=True, capture_output=True)
        return out.read_text()

    with ThreadPoolExecutor(len(DECODE_INST)) as ex:
        return "\n".join(ex.map(compile_one, enumerate(DECODE_INST)))


def test_the_windowed_decode_keeps_the_decode_s_rules(asm):
    """m0 and LDS loads, the merge's device-scope accesses, and an MFMA's wait states: test_isa.py has the reasons."""
    assert len(isa.kernels(asm)) >= 30
    isa.test_m0_is_only_the_lds_load_base(asm)
    isa.test_every_lds_load_is_ours(asm)
    isa.test_split_merge_is_device_scope_accesses_without_cache_maintenance(asm)
    isa.test_mfma_results_keep_their_wait_states_on_every_path(asm)


# ------------------------------------------------------------------ the native host side
SCRIPT = r"""
import ctypes, importlib.util, sys
import torch
spec = importlib.util.spec_from_file_location("_stepcall", sys.argv[1])
m = importlib.util.module_from_spec(spec)
spec.loader.exec_module(m)
sys.path.insert(0, sys.argv[2])
from kushkash_amd import _lib
calls, keep, errors = [], [], []
def entry(name):
    sig = (_lib.WINDOW_SIGNATURES | _lib.STEP_SIGNATURES)[name]
    size = name == "kush_sample_scratch"
    f = ctypes.CFUNCTYPE(ctypes.c_int64 if size else ctypes.c_int, *sig)(
        (lambda r, v: 4096) if size else (lambda *a: calls.append((name, a)) or code[0]))
    keep.append(f)
    return ctypes.cast(f, ctypes.c_void_p).value
code = [0]
def check(name, rc):
    errors.append((name, rc))
    raise RuntimeError(name)
m.bind(check, *(entry(n) for n in ("kush_window_decode", "kush_window_attend", "kush_block_table", "kush_step_maps",
                                   "kush_sample", "kush_sample_scratch")))
S, H, G, D, B, V = 3, 2, 4, 64, 5, 200
i32 = dict(dtype=torch.int32)
sync = torch.zeros(64, **i32)
t = dict(k=torch.randn(S, H, D), v=torch.randn(S, H, D), q=torch.randn(S, H * G, D), out=torch.zeros(S, H * G, D),
         cache=torch.zeros(B, H, 2560, dtype=torch.uint8), table=torch.zeros(S, 2, **i32), lens=torch.ones(S, **i32),
         tidx=torch.arange(S, **i32), tail=torch.zeros(S, H, 32, D), work=torch.zeros(S * H * 2 * G * (D + 2)), order=torch.arange(S, **i32),
         rq=torch.randn(7, H * G, D).half(), rk=torch.randn(20, H, D).half(), rv=torch.randn(20, H, D).half(), ro=torch.zeros(7, H * G, D).half(),
         cq=torch.tensor([0, 3, 7], **i32), ck=torch.tensor([0, 12, 20], **i32),
         map=torch.zeros(6, 64, **i32), req=torch.arange(S, **i32), tt=torch.zeros(S, 2, **i32), tl=torch.zeros(S, **i32), ts=torch.zeros(S, **i32),
         new=torch.ones(S, **i32), old=torch.ones(S, **i32), slots=torch.arange(S, **i32),
         x=torch.randn(S, V), u=torch.rand(S), temp=torch.ones(S), topk=torch.ones(S, **i32), topp=torch.ones(S), minp=torch.ones(S),
         tok=torch.zeros(S, dtype=torch.int64))
def decode(x, ns=2):
    return m.decode(D, 4, G, 0, 0, sync.data_ptr(), 64, x["k"], x["v"], x["q"], x["out"], x["cache"], x["table"], x["lens"], x["tidx"],
                    x["tail"], 0.1, ns, x["work"], 4, x["order"], False, 9, 2, 0)
def alone(x):
    return decode(dict(x, k=None, v=None), 1)
def attend(x):
    return m.attend(x["rq"], x["rk"], x["rv"], x["ro"], x["cq"], x["ck"], 0.1, 9, 2, 4, 12, 4, 0, 0, 2, 2, 0)
def table(x):
    return m.block_table(x["map"], x["req"], x["lens"], 2, (x["tt"], x["tl"], x["ts"]), 0)
def maps(x):
    return m.step_maps(x["new"], x["old"], x["slots"], x["table"], (S, S, 2 * S, S, 0, S, 0, 0), 0)
def sample(x):
    return m.sample(x["x"], x["u"], x["temp"], x["topk"], x["topp"], x["minp"], x["tok"], 0)

CALLS = [(decode, "k v q out cache table lens tidx tail work order"), (alone, "q out cache table lens tidx tail order"),
         (attend, "rq rk rv ro cq ck"), (table, "map req lens tt tl ts"), (maps, "new old slots table"),
         (sample, "x u temp topk topp minp tok")]
for fn, names in CALLS:
    assert fn(t) is not None and len(calls) == 1, fn.__name__      # the plain call is taken ...
    want = {t[n].data_ptr() for n in names.split()}
    assert want <= set(calls.pop()[1]), fn.__name__                # ... with every tensor's address,
    for n in names.split():                                        # and none without one,
        print(fn.__name__, n, flush=True)
        def body(x):
            assert type(x) is torch.Tensor
            assert fn(dict(t, **{n: x})) is None
            return torch.zeros(1)
        torch.vmap(body)(t[n][None])
        for other in (None if n not in ("order", "ro", "tok") else 5, t[n].double(), t[n][:1] if t[n].shape[0] > 1 else t[n][:0]):
            if (other is None and n in ("k", "work")) or n == "cache" or (n in ("map", "tail") and other is not None
                                                                             and other.dtype == t[n].dtype):
                continue                                           # (a cache may be of any type, a map and tails of any rows)
            assert fn(dict(t, **{n: other})) is None, n            # nor one of another kind or size
    assert not calls
    code[0] = -2                                                   # a refusal of the library raises
    try:
        fn(t)
        raise SystemExit("no error")
    except RuntimeError:
        pass
    code[0] = 0
    assert len(errors) == 1 and errors.pop()[1] == -2
    calls.clear()
for bad in (lambda: m.sample(t["x"], t["u"], -1.0, 0, 1.0, 0.0, None, 0), lambda: m.sample(t["x"], t["u"], 1.0, -1, 1.0, 0.0, None, 0),
            lambda: m.sample(t["x"], t["u"], 1.0, 1.0, 1.0, 0.0, None, 0), lambda: m.sample(t["x"], t["u"], 1.0, 0, float("nan"), 0.0, None, 0),
            lambda: m.sample(t["x"].requires_grad_(), t["u"], 1.0, 0, 1.0, 0.0, None, 0),
            lambda: m.block_table(t["map"], t["req"], t["lens"], -1, None, 0), lambda: m.block_table(t["map"], t["req"], t["lens"], True, None, 0),
            lambda: m.step_maps(t["new"], t["old"], t["slots"], t["table"], (S, -1, 0, 0, 0, 0, 0, 0), 0),
            lambda: m.attend(t["rq"], t["rk"], t["rv"], None, t["cq"], t["ck"], 0.0, 9, 2, 4, 12, 4, 0, 0, 2, 2, 0),
            lambda: m.attend(t["rq"], t["rk"], t["rv"], None, t["cq"], t["ck"], 0.1, 0, 2, 4, 12, 4, 0, 0, 2, 2, 0)):
    assert bad() is None and not calls
print("every call answered")
"""


@pytest.fixture(scope="module")
def stepcall(tmp_path_factory):
    """Built without its device checks."""
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    import importlib
    build = importlib.import_module("kushkash_amd.build")
    tmp = tmp_path_factory.mktemp("stepcall")
    src = (build.PKG / "csrc" / build.STEP_SOURCE).read_text()
    for check, put in (("t.is_cuda() && ", ""), ("    need(t.get_device() == impl->getDevice().index());\n    return t.get_device();", "    return 0;"),
                       ("need(t.get_device() == d);", ""), ("dev == integer(a[4], 0, 127) && out.get_device() == dev && cache.get_device() == dev && "
                                                            "tail.get_device() == dev", "true"),
                       ("need(k.get_device() == dev && v.get_device() == dev && ", "need("), ("need(out.get_device() == dev && ", "need("),
                       ("    static const c10::impl::DeviceGuardImplInterface* const impl = c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA);\n", "")):
        assert src.count(check) == 1, check
        src = src.replace(check, put)
    (tmp / build.STEP_SOURCE).write_text(src)
    out = tmp / "_stepcall.so"
    cmd = build.fastcall_command(out, build.STEP_SOURCE)
    at = cmd.index(str(build.PKG / "csrc" / build.STEP_SOURCE))
    subprocess.run([*cmd[:at], str(tmp / build.STEP_SOURCE), *cmd[at + 1:]], check=True, capture_output=True)
    return out


def test_what_the_native_calls_take(stepcall, tmp_path):
    (tmp_path / "calls.py").write_text(SCRIPT)
    r = subprocess.run([sys.executable, str(tmp_path / "calls.py"), str(stepcall), str(Path(kushkash_amd.__file__).parent.parent)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "every call answered" in r.stdout, (r.returncode, r.stdout[-300:], r.stderr[-2000:])


def test_an_extension_of_another_abi_is_refused(monkeypatch):
    for old in (types.SimpleNamespace(), types.SimpleNamespace(ABI=_lib.ABI_VERSION - 1)):
        monkeypatch.setitem(sys.modules, "kushkash_amd._stepcall", old)
        monkeypatch.setattr(kushkash_amd, "_stepcall", old, raising=False)
        _lib.stepcall.cache_clear()
        with pytest.raises(RuntimeError, match=f"expected {_lib.ABI_VERSION}; rebuild it"):
            _lib.stepcall()
    monkeypatch.undo()
    _lib.stepcall.cache_clear()
    assert _lib.stepcall() is None or _lib.stepcall().ABI == _lib.ABI_VERSION


def test_the_native_calls_step_aside_where_launches_are_recorded(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda name, *args: None)
    assert _lib.native() is None
