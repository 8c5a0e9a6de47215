"""What the chunked path over the paged cache refuses, before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

from subspec_b200 import _lib
from subspec_b200.attention import append_paged_kv_slots, chunk_attention_paged, window_attention_paged
from subspec_b200.pages import DevicePagePool


def _pool(dtype=torch.bfloat16, D=64):
    return torch.zeros(2, 6, 2, 8, 2, D, dtype=dtype)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _call(fn=chunk_attention_paged, **kw):
    args = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), pool=_pool(), layer=0,
                page_table=torch.zeros(2, 3, dtype=torch.int32), kv_len=_i32(5, 4), q_indptr=_i32(0, 2, 3))
    args.update(kw)
    return fn(args.pop("q"), args.pop("pool"), args.pop("layer"), **args)


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(3, 4, 64)),                                           # type
    dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)),                      # another type than the pool's
    dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)),                     # heads not a multiple
    dict(q=torch.zeros(3, 0, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16)),                  # a batch axis
    dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)),                     # head_dim
    dict(q=torch.zeros(3, 4, 96, dtype=torch.bfloat16), pool=_pool(D=96)),
    dict(pool=_pool()[:, :, :1]),                                            # no V plane
    dict(pool=_pool()[:, ::2]),                                              # pool not contiguous
    dict(layer=2), dict(layer=-1),
    dict(page_table=torch.zeros(2, 3, dtype=torch.int64)),
    dict(page_table=torch.zeros(2, 6, dtype=torch.int32)[:, ::2]),
    dict(kv_len=_i32(5, 4, 3)), dict(kv_len=torch.tensor([5, 4])),
    dict(q_indptr=_i32(0, 2)), dict(q_indptr=torch.tensor([0, 2, 3])),
    dict(out=torch.zeros(3, 4, 64)), dict(out=torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
    dict(out=torch.zeros(3, 4, 65, dtype=torch.bfloat16)[..., 1:]),          # rows not 16-byte aligned
    dict(max_q_len=-1), dict(status=torch.zeros(1, dtype=torch.int64)),
])
def test_attention_refusals(bad):
    with pytest.raises(ValueError):
        _call(**bad)


@pytest.mark.parametrize("out", [torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, 4, 64),
                                 torch.zeros(3, 1, 64, dtype=torch.bfloat16).expand(3, 4, 64)])
def test_output_rows_that_share_memory_are_refused(out):
    with pytest.raises(ValueError, match="share memory"):  # by its words: host tensors are refused in the end anyway
        _call(out=out)


@pytest.mark.parametrize("bad", [dict(window=0), dict(window=-3), dict(window=4, sinks=-1)])
def test_window_refusals(bad):
    with pytest.raises(ValueError):
        _call(window_attention_paged, **bad)


@pytest.mark.parametrize("bad", [
    dict(k=torch.zeros(3, 2, 64)), dict(k=torch.zeros(2, 2, 64, dtype=torch.bfloat16)),
    dict(k=torch.zeros(3, 1, 64, dtype=torch.bfloat16), v=torch.zeros(3, 1, 64, dtype=torch.bfloat16)),
    dict(slot_map=torch.zeros(3, dtype=torch.int32)), dict(slot_map=torch.zeros(2, dtype=torch.int64)),
    dict(slot_map=torch.zeros(6, dtype=torch.int64)[::2]), dict(layer=5), dict(pool=_pool().float()),
])
def test_append_refusals(bad):
    args = dict(pool=_pool(), layer=1, k=torch.zeros(3, 2, 64, dtype=torch.bfloat16),
                v=torch.zeros(3, 2, 64, dtype=torch.bfloat16), slot_map=torch.zeros(3, dtype=torch.int64))
    args.update(bad)
    with pytest.raises(ValueError):
        append_paged_kv_slots(args["pool"], args["layer"], args["k"], args["v"], slot_map=args["slot_map"])


def test_plan_refusals():
    with pytest.raises(ValueError):
        DevicePagePool(2, 8, 4, 4, "cpu").plan_chunks(_i32(1, 1))             # no room for a token list
    pool = DevicePagePool(2, 8, 4, 4, "cpu", max_append=8)
    for bad in (dict(n_new=_i32(1)), dict(n_new=torch.tensor([1.0, 2.0])), dict(n_new=_i32(1, 1), set_len=_i32(1, 2, 3))):
        with pytest.raises(ValueError):
            pool.plan_chunks(bad["n_new"], set_len=bad.get("set_len"))


def test_host_tensors_are_refused(cuda_lib):
    """There is no CPU form: calls that are right in all else, on host tensors."""
    for call in (lambda: _call(), lambda: _call(window_attention_paged, window=3),
                 lambda: append_paged_kv_slots(_pool(), 0, torch.zeros(3, 2, 64, dtype=torch.bfloat16),
                                               torch.zeros(3, 2, 64, dtype=torch.bfloat16), slot_map=torch.arange(3)),
                 lambda: DevicePagePool(2, 8, 4, 4, "cpu", max_append=8).plan_chunks(_i32(1, 1))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_c_entry_points_check_their_arguments(cuda_lib):
    """Struct sizes, enums, null pointers and unsupported shapes: refused before any launch; empty calls pass."""
    p = _lib.ChunkPlanArgs()
    assert cuda_lib.subspec_chunk_plan(C.byref(p), None) == _lib.EINVAL
    p.struct_size = C.sizeof(_lib.ChunkPlanArgs)
    p.batch, p.num_pages, p.page_len, p.pages_per_seq = 2, 8, 4, 4
    assert cuda_lib.subspec_chunk_plan(C.byref(p), None) == _lib.EINVAL       # null pointers
    for name in ("free_mask", "page_table", "n_pages", "kv_len", "n_new", "q_indptr"):
        setattr(p, name, 16)
    p.max_tokens = 4
    assert cuda_lib.subspec_chunk_plan(C.byref(p), None) == _lib.EINVAL       # no token outputs
    p.max_tokens, p.pages_per_seq, p.page_len = 0, 1 << 20, 1 << 12
    assert cuda_lib.subspec_chunk_plan(C.byref(p), None) == _lib.EUNSUPPORTED  # positions pass 32 bits
    p.pages_per_seq, p.page_len, p.num_pages = 4, 4, 1 << 24
    assert cuda_lib.subspec_chunk_plan(C.byref(p), None) == _lib.EUNSUPPORTED  # more pages than shared memory counts
    s = _lib.KvAppendSlotsArgs()
    assert cuda_lib.subspec_kv_append_slots(C.byref(s), None) == _lib.EINVAL
    s.struct_size = C.sizeof(_lib.KvAppendSlotsArgs)
    s.num_kv_heads, s.head_dim, s.layers, s.num_pages, s.page_len = 2, 64, 1, 8, 4
    assert cuda_lib.subspec_kv_append_slots(C.byref(s), None) == _lib.OK
    s.tokens = 3
    assert cuda_lib.subspec_kv_append_slots(C.byref(s), None) == _lib.EINVAL
    s.k_token_stride = 12
    assert cuda_lib.subspec_kv_append_slots(C.byref(s), None) == _lib.EUNSUPPORTED
    a = _lib.ChunkAttnArgs()
    n = C.c_size_t(0)
    assert cuda_lib.subspec_chunk_attention_paged(C.byref(a), None) == _lib.EINVAL
    assert cuda_lib.subspec_chunk_attention_scratch_bytes(C.byref(a), C.byref(n)) == _lib.EINVAL
    a.struct_size = C.sizeof(_lib.ChunkAttnArgs)
    a.num_q_heads, a.num_kv_heads, a.head_dim, a.layers, a.num_pages, a.page_len, a.pages_per_seq = 4, 2, 64, 1, 8, 4, 4
    a.dtype, a.sm_scale = _lib.BF16, 0.125
    assert cuda_lib.subspec_chunk_attention_paged(C.byref(a), None) == _lib.OK  # an empty batch
    a.batch, a.tokens, a.max_q_len = 2, 3, 2
    assert cuda_lib.subspec_chunk_attention_paged(C.byref(a), None) == _lib.EINVAL  # null pointers
    assert cuda_lib.subspec_chunk_attention_scratch_bytes(C.byref(a), C.byref(n)) == _lib.OK
    for name, bad, rc in (("sm_scale", 0.0, _lib.EINVAL), ("sm_scale", float("nan"), _lib.EINVAL), ("dtype", 7, _lib.EINVAL),
                          ("window", -1, _lib.EINVAL), ("sinks", -1, _lib.EINVAL), ("layer", 1, _lib.EINVAL),
                          ("head_dim", 80, _lib.EUNSUPPORTED),
                          ("num_q_heads", 3, _lib.EUNSUPPORTED)):
        old = getattr(a, name)
        setattr(a, name, bad)
        assert cuda_lib.subspec_chunk_attention_paged(C.byref(a), None) == rc, name
        setattr(a, name, old)


def test_argument_structs_match_the_header(tmp_path):
    """Sizes and offsets of the three argument structs as a C99 compiler lays them out."""
    import subprocess
    from pathlib import Path

    include = Path(__file__).resolve().parent.parent / "include"
    structs = {"subspec_chunk_plan_args": _lib.ChunkPlanArgs, "subspec_kv_append_slots_args": _lib.KvAppendSlotsArgs,
               "subspec_chunk_attn_args": _lib.ChunkAttnArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "subspec_b200.h"', "int main(void) {"]
    for cname, mirror in structs.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(include), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                                        text=True).stdout.splitlines())
    for cname, mirror in structs.items():
        assert int(got[cname]) == C.sizeof(mirror)
        for f, _ in mirror._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(mirror, f).offset, (cname, f)


def test_the_status_word_belongs_to_a_device(cuda_lib):
    from subspec_b200.attention import check_status

    with pytest.raises(ValueError, match="CUDA"):
        check_status("cpu")
    assert cuda_lib.subspec_default_status(None) == _lib.EINVAL
