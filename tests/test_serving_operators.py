"""What the serving operators refuse or lay out without a GPU: the argument structures of the C ABI
against the header, null and inconsistent arguments at the C entries, and the host side of a batch
with shared prefixes."""

import ctypes as C
import pathlib
import subprocess

import pytest
import torch

from latent_attn import MLAConfig, SharedPrefixBatch, _lib

HEADER = pathlib.Path(__file__).resolve().parents[1] / "include"

STRUCTS = {"mla_append_rope_args_t": _lib.MlaAppendRopeArgs, "mla_prefix_args_t": _lib.MlaPrefixArgs,
           "mla_lora_args_t": _lib.MlaLoraArgs}


def test_struct_layouts_match_the_header(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        for field, _ in cls._fields_:
            lines.append(f'printf(" %zu", offsetof({name}, {field}));')
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"latent_attn_b200/mla.h\"\nint main(void) {\n" +
                   "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    cuda = pathlib.Path("/usr/local/cuda/include")
    subprocess.run(["gcc", "-I", str(HEADER), "-I", str(cuda), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, *offsets = line.split()
        cls = STRUCTS[name]
        assert C.sizeof(cls) == int(size), name
        assert [getattr(cls, f).offset for f, _ in cls._fields_] == [int(o) for o in offsets], name


def _cfg():
    return _lib.MlaConfig(512, 512, 128, 64, 16, 128)


def _refused(call):
    with pytest.raises(_lib.MlaError):
        _lib.check(call())


def test_entries_refuse_null_and_bad_arguments():
    lib, cfg = _lib.load(), _cfg()
    _refused(lambda: lib.mla_cache_append_rope(C.byref(cfg), None, None))
    _refused(lambda: lib.mla_cache_append_rope(None, C.byref(_lib.MlaAppendRopeArgs()), None))
    _refused(lambda: lib.mla_cache_append_rope(C.byref(cfg), C.byref(_lib.MlaAppendRopeArgs()), None))
    _refused(lambda: lib.mla_prefix_decode(C.byref(cfg), None, None, 0, None))
    _refused(lambda: lib.mla_prefix_decode(C.byref(cfg), C.byref(_lib.MlaPrefixArgs()), None, 0, None))
    _refused(lambda: lib.mla_linear_lora(None, None, 0, None))
    _refused(lambda: lib.mla_linear_lora(C.byref(_lib.MlaLoraArgs()), None, 0, None))


@pytest.mark.parametrize("m,adapters,rank", [(1 << 23, 256, 8), (1 << 23, 128, 128), (1 << 24, 1, 8), (1, 1, 264),
                                             (1, 1, 12), (1, 0, 8), (0, 1, 8)])
def test_projection_refuses_sizes_before_it_looks_at_memory(m, adapters, rank):
    lib = _lib.load()
    a = _lib.MlaLoraArgs(1, m, 64, 64, 16, 0, 16, adapters, rank, 16, 16, 16, None, 16)
    size = C.c_size_t()
    with pytest.raises(_lib.MlaError, match="tokens|rank|M must|num_adapters|positive"):
        _lib.check(lib.mla_linear_lora_workspace_size(C.byref(a), C.byref(size)))


def test_shared_prefix_batch_lays_out_positions():
    cfg = MLAConfig(512, 512, 128, 64, 16, 128)
    b = SharedPrefixBatch(cfg, "cpu", [2, 1], [100, 0], [3, 0, 7], 10, prefix_offsets=[0, 0], own_offsets=[200, 220, 240])
    assert b.group_starts.tolist() == [0, 2, 3] and b.positions.tolist() == [103, 100, 7]
    assert b.row_offsets.tolist() == [100, 120, 240] and b.row_offsets.dtype == torch.int64
    b._next.copy_(b.positions + 1)
    b.advance()
    assert b.positions.tolist() == [104, 101, 8] and b.own_lens.tolist() == [4, 1, 8]
    p = SharedPrefixBatch(cfg, "cpu", [2, 1], [128, 64], [3, 0, 7], 64, prefix_table=[[9, 8], [7, 0]],
                          own_table=[[1], [2], [3]], page_rows=64)
    assert p.row_table.tolist() == [[0, 0, 1], [0, 0, 2], [0, 3, 0]]


@pytest.mark.parametrize("kw,what", [
    (dict(prefix_lens=[1]), "one entry per group"),
    (dict(own_lens=[0]), "one entry per group"),
    (dict(max_own_len=2), "max_own_len"),
    (dict(prefix_offsets=None), "prefix_offsets and own_offsets"),
    (dict(page_rows=64), "prefix_offsets and own_offsets"),
    (dict(page_rows=64, prefix_offsets=None, own_offsets=None, prefix_table=[[0, 1], [2, 3]],
          own_table=[[4], [5], [6]]), "multiples of page_rows"),
])
def test_shared_prefix_batch_refusals(kw, what):
    args = dict(group_sizes=[2, 1], prefix_lens=[100, 0], own_lens=[3, 0, 7], max_own_len=10, prefix_offsets=[0, 0],
                own_offsets=[200, 220, 240])
    args.update(kw)
    with pytest.raises(RuntimeError, match=what):
        SharedPrefixBatch(MLAConfig(512, 512, 128, 64, 16, 128), "cpu", **args)
