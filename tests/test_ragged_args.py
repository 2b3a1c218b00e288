"""What the ragged-batch entry points refuse, checked without a GPU: every
argument check runs before the engine is asked for, and device addresses are
never read on the host."""
import pytest

from burn_rocket_b200 import _lib

P = 0x7000_0000_0000  # a 16-byte aligned address that nothing on the host reads


def call(name, base, **change):
    args = dict(base)
    assert set(change) <= set(args), change
    args.update(change)
    packer = {"rb_kv_append": _lib.KV_APPEND_ARGS, "rb_attention_paged": _lib.ATTENTION_PAGED_ARGS,
              "rb_attention_packed": _lib.ATTENTION_PACKED_ARGS}[name]
    return getattr(_lib.load(), name)(packer.pack(*(0 if v is None else v for v in args.values())), None)


# In the order of the C structures.
APPEND = dict(q=P, k=P + 64, v=P + 128, ldq=2048, ldk=1024, ldv=1024, tokens=8, batch=2, cu=P, kv_len=P, q_norm=P,
              k_norm=None, cos=P, sin=P, max_pos=100, q_out=P + 256, ldq_out=2048, k_cache=P, v_cache=P,
              page_stride=16 * 1024, num_pages=10, table=P, ld_table=4, dtype=1, n_head=16, n_kv_heads=8, head_dim=128,
              page_size=16, eps=1e-6)
PAGED = dict(q=P + 64, out=P + 256, k_cache=P, v_cache=P, ldq=2048, ldo=2048, tokens=8, batch=2, cu=P, kv_len=P, max_q=4,
             max_kv=0, page_stride=16 * 1024, num_pages=10, table=P, ld_table=4, window=-1, dtype=2, n_head=16,
             n_kv_heads=8, head_dim=128, page_size=16, scale=0.1, softcap=0.0)
PACKED = dict(q=P, k=P + 64, v=P + 128, out=P + 256, ldq=4096, ldk=4096, ldv=4096, ldo=2048, tokens=8, batch=2, cu=P,
              window=-1, dtype=1, n_head=16, n_kv_heads=8, head_dim=128, mode=2, scale=0.1, softcap=0.0)
NAN, INF = float("nan"), float("inf")

COMMON = [dict(dtype=0), dict(dtype=3), dict(tokens=-1), dict(batch=-1), dict(tokens=1 << 31), dict(n_head=15),
          dict(n_head=0), dict(n_kv_heads=0), dict(n_head=-16), dict(n_head=2048, n_kv_heads=8), dict(cu=None)]
CACHE = [dict(page_size=8), dict(page_size=48), dict(page_size=256), dict(page_size=0), dict(num_pages=0),
         dict(ld_table=0), dict(table=None), dict(page_stride=16 * 1024 - 8), dict(page_stride=16 * 1024 + 4),
         dict(k_cache=None), dict(v_cache=None), dict(k_cache=P + 8), dict(v_cache=P + 2), dict(head_dim=72),
         dict(head_dim=96), dict(kv_len=None)]
SOFTMAX = [dict(scale=0.0), dict(scale=-0.1), dict(scale=NAN), dict(scale=INF), dict(softcap=-1.0), dict(softcap=NAN),
           dict(softcap=INF)]


@pytest.mark.parametrize("change", COMMON + CACHE + [
    dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(ldq=2040), dict(ldk=1020), dict(ldv=1028),
    dict(q=P + 8), dict(k=P + 2), dict(q_out=P + 4), dict(cos=None), dict(sin=None), dict(cos=P + 4), dict(q_norm=P + 8),
    dict(max_pos=0), dict(eps=NAN), dict(eps=-1.0), dict(q_out=P, ldq=4096)])  # in place with two strides
def test_kv_append_refuses(change):
    rc = call("rb_kv_append", APPEND, **change)
    assert rc in (_lib.RB_E_SHAPE, _lib.RB_E_UNSUPPORTED), (rc, change)
    assert _lib.last_error().startswith("kv_append:")


@pytest.mark.parametrize("change", COMMON + CACHE + SOFTMAX + [
    dict(q=None), dict(out=None), dict(ldq=1024), dict(ldo=2044), dict(q=P + 2), dict(out=P + 8), dict(out=P + 64),
    dict(out=P), dict(max_q=-1), dict(max_kv=-1)])
def test_attention_paged_refuses(change):
    rc = call("rb_attention_paged", PAGED, **change)
    assert rc in (_lib.RB_E_SHAPE, _lib.RB_E_UNSUPPORTED), (rc, change)
    assert _lib.last_error().startswith("attention_paged:")


@pytest.mark.parametrize("change", COMMON + SOFTMAX + [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(ldk=1000), dict(ldv=4092), dict(v=P + 4),
    dict(out=P), dict(out=P + 64), dict(out=P + 128), dict(mode=1), dict(mode=5), dict(mode=6), dict(mode=7),
    dict(mode=-1), dict(head_dim=80), dict(head_dim=0)])
def test_attention_packed_refuses(change):
    rc = call("rb_attention_packed", PACKED, **change)
    assert rc in (_lib.RB_E_SHAPE, _lib.RB_E_UNSUPPORTED), (rc, change)
    assert _lib.last_error().startswith("attention_packed:")


def test_null_arguments_are_refused():
    for name in ("rb_kv_append", "rb_attention_paged", "rb_attention_packed"):
        assert getattr(_lib.load(), name)(None, None) == _lib.RB_E_SHAPE


@pytest.mark.parametrize("name,base", [("rb_kv_append", APPEND), ("rb_attention_paged", PAGED),
                                       ("rb_attention_packed", PACKED)])
def test_empty_batches_are_no_work(name, base):
    assert call(name, base, tokens=0) == _lib.RB_OK
    assert call(name, base, batch=0) == _lib.RB_OK


def test_argument_structures_match_the_header(tmp_path):
    """The packed layouts are the C compiler's."""
    import subprocess
    import struct
    from pathlib import Path
    header = Path(__file__).resolve().parent.parent / "include" / "rocket_b200.h"
    src = tmp_path / "layout.c"
    src.write_text(f'''#include <stdio.h>
#include <stddef.h>
#include "{header}"
int main(void) {{
  printf("%zu %zu %zu\\n", sizeof(rb_kv_append_args), sizeof(rb_attention_paged_args), sizeof(rb_attention_packed_args));
  printf("%zu %zu %zu\\n", offsetof(rb_kv_append_args, eps), offsetof(rb_attention_paged_args, softcap),
         offsetof(rb_attention_packed_args, softcap));
}}''')
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "layout")], check=True)
    sizes, last = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()
    packers = (_lib.KV_APPEND_ARGS, _lib.ATTENTION_PAGED_ARGS, _lib.ATTENTION_PACKED_ARGS)
    assert [p.size - 4 for p in packers] == [int(x) for x in last.split()]
    assert [(p.size + 7) // 8 * 8 for p in packers] == [int(x) for x in sizes.split()]
    assert struct.calcsize("P") == 8


def test_good_arguments_need_the_engine():
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch on addresses that are not memory")
    for name, base in (("rb_kv_append", APPEND), ("rb_attention_paged", PAGED), ("rb_attention_packed", PACKED)):
        assert call(name, base) == _lib.RB_E_IO
        assert "rb_init" in _lib.last_error()


def test_python_refusals():
    """The wrappers' own checks: shapes, dtypes, strides and devices."""
    import torch
    import burn_rocket_b200 as rb
    q = torch.zeros(4, 256, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(rb.OpFailure, match="CUDA"):
        rb.attention_packed(q, q, q, cu, 2, 2, 128, 0.1)
    with pytest.raises(rb.OpFailure, match="CUDA"):
        rb.kv_append(q, q, q, q, q, cu, cu, cu, 2, 2, 128, q, q)
    with pytest.raises(rb.OpFailure, match="CUDA"):
        rb.attention_paged(q, q, q, cu, cu, cu, 2, 2, 128, 0.1, max_q=4)


@pytest.mark.parametrize("name,base", [("rb_kv_append", APPEND), ("rb_attention_paged", PAGED)])
@pytest.mark.parametrize("empty", [dict(batch=0), dict(tokens=0)])
def test_empty_batches_need_no_table(name, base, empty):
    """An empty tensor has no address: that of an empty batch is not asked for."""
    assert call(name, base, table=None, **empty) == _lib.RB_OK
    assert call(name, base, table=None, ld_table=0, **empty) == _lib.RB_OK


@pytest.mark.parametrize("where", ["k", "v", "k_cache", "v_cache"])
def test_rotated_queries_over_another_input_are_refused(where):
    """q may be rotated in place; over k or v other heads would read what was
    written, over the cache other tokens' slots would be lost."""
    base = dict(APPEND, n_kv_heads=16, ldk=2048, ldv=2048, page_stride=16 * 2048, k_cache=P + 512, v_cache=P + 1024)
    assert call("rb_kv_append", base, q_out=base[where]) == _lib.RB_E_SHAPE
    assert _lib.last_error().startswith("kv_append: q_out")
