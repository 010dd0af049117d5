"""The serving operators' refusals (include/vitna_serve.h), which need no GPU: what the host can see is checked before
any pointer is looked at, and a pointer that is no device memory is refused. No kernel is launched here."""
import ctypes as C
import os
import re

import pytest

import vitna_amd as va

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ERR = C.create_string_buffer(512)
HOST = (C.c_char * 4096)()
AT = (C.addressof(HOST) + 255) & ~255


def view(**kw):
    d = dict(k=AT, v=AT, dtype=va.F32, n_heads=8, n_kv_heads=2, head_dim=128, ctx=64, seqs=3)
    d.update(kw)
    return va.kv_view(**d)


def refused(call, text):
    with pytest.raises(va.VitnaError) as e:
        call()
    assert re.search(text, str(e.value)), str(e.value)


def test_library_exports_every_declared_function():
    with open(os.path.join(ROOT, "include", "vitna_serve.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(vitna_hip_\w+)\s*\(", text)))
    assert len(names) >= 7
    for n in names:
        assert getattr(va.hip(), n) is not None


VIEWS = [
    (dict(dtype=va.Q8_0), "dtype"), (dict(head_dim=96), "dimensions"), (dict(n_heads=7), "query heads"), (dict(n_heads=34), "query heads"),
    (dict(n_kv_heads=0, n_heads=0, pos_stride=256), "key-value heads"), (dict(n_heads=0), "query heads"), (dict(ctx=0), "positions"),
    (dict(ctx=(1 << 30) + 1), "positions"), (dict(seqs=0), "sequences"), (dict(seqs=1 << 31), "sequences"),
    (dict(pos_stride=258), "strides"), (dict(dtype=va.BF16, head_stride=132), "strides"), (dict(seq_stride=1 << 60), "too large"), (dict(pos_stride=(1 << 23) + 4), "positions 8388612 elements apart"),
    (dict(k=AT + 4), "aligned"), (dict(v=AT + 8), "aligned"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"),
]


@pytest.mark.parametrize("change,text", VIEWS, ids=[str(i) for i in range(len(VIEWS))])
def test_views_refused(change, text):
    v = view(**change)
    refused(lambda: va.attention_rows(v, AT, AT, 1, AT, AT, 1 << 30), text)
    refused(lambda: va.attention_run(v, 0, 0, AT, 1, AT, AT, 1 << 30), text)
    refused(lambda: va.attention_rows_work(v, 1), "not served") if "aligned" not in text else None
    if text not in ("query heads", "scale"):
        refused(lambda: va.kv_reorder(v, 1, 0, AT, AT, AT, 1, 2), text)


def test_attention_arguments_refused():
    v = view()
    work = va.attention_rows_work(v, 5)
    assert work > 0 and va.attention_run_work(v, 0, 64) > 0
    refused(lambda: va.attention_rows(v, AT, AT, 0, AT, AT, 1 << 30), "rows")
    refused(lambda: va.attention_rows(v, AT, AT, 65536, AT, AT, 1 << 40), "rows")
    refused(lambda: va.attention_rows(v, AT, 0, 1, AT, AT, 1 << 30), "rows is missing")
    refused(lambda: va.attention_rows(v, AT, AT, 5, AT, AT, work - 1), "bytes of work")
    refused(lambda: va.attention_rows(v, AT + 4, AT, 5, AT, AT, work), "aligned")
    refused(lambda: va.attention_rows(v, AT, AT + 4, 5, AT, AT, work), "aligned")
    refused(lambda: va.attention_rows(v, AT, AT, 5, AT, AT, work, out_stride=1020), "floats apart")
    refused(lambda: va.attention_rows(v, AT, AT, 5, AT, AT, work, out_stride=1028), "out is q")
    refused(lambda: va.attention_run(v, 0, 0, AT, 5, AT, AT, 1 << 20, q_stride=2048), "out is q")
    refused(lambda: va.attention_rows(v, AT, AT, 5, AT, AT, work, q_stride=1025), "floats apart")
    refused(lambda: va.attention_rows(v, AT, AT, 5, AT, AT, work), "not device memory")
    refused(lambda: va.attention_rows(view(k=None), AT, AT, 5, AT, AT, work), "k is missing")
    refused(lambda: va.attention_run(v, 3, 0, AT, 1, AT, AT, 1 << 30), "sequence 3")
    refused(lambda: va.attention_run(v, 0, 60, AT, 5, AT, AT, 1 << 30), "positions 60")
    refused(lambda: va.attention_run(v, 0, 65, AT, 1, AT, AT, 1 << 30), "positions 65")
    refused(lambda: va.attention_run(v, 0, 0, AT, 0, AT, AT, 1 << 30), "rows")
    refused(lambda: va.attention_run(v, 0, 0, AT, 1, AT, AT, 1 << 30), "not device memory")
    refused(lambda: va._call(va.hip().vitna_hip_attention_rows, None, AT, 0, AT, 1, 0, 0, AT, 0, AT, 1 << 30, 0), "no cache")


def select(**kw):
    d = dict(logits=AT, vocab=100, groups=1, width=2, keep=2, scores=AT, best=AT, parents=AT, tokens=AT, work=AT, work_bytes=1 << 30)
    d.update(kw)
    return lambda: va.beam_select(**d)


@pytest.mark.parametrize("change,text", [
    (dict(groups=0), "groups"), (dict(groups=65536), "groups"), (dict(width=0), "beams"), (dict(width=65), "beams"), (dict(keep=0), "results"),
    (dict(keep=65), "results"), (dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 24) + 1), "vocabulary"), (dict(stride=99), "floats apart"),
    (dict(ended=AT, end_token=100), "outside"), (dict(ended=AT, end_token=-1), "outside"), (dict(logits=AT + 2), "aligned"),
    (dict(work=AT + 4), "aligned"), (dict(work_bytes=8), "bytes of work"), (dict(logits=0), "logits is missing"), (dict(), "not device memory"),
])
def test_selections_refused(change, text):
    refused(select(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(groups=0), "groups"), (dict(width=0), "beams"), (dict(width=65), "beams"), (dict(layers=0), "layers"), (dict(layers=32768), "layers"),
    (dict(layers=2, layer_stride=8192), "overlap"), (dict(layers=2, layer_stride=64 * 256 * 3 - 4), "overlap"),
    (dict(layers=2, layer_stride=2), "elements apart"), (dict(seqs=AT + 2), "aligned"), (dict(spans=0), "not device memory"),
])
def test_reorders_refused(change, text):
    d = dict(layers=1, layer_stride=0, seqs=AT, parents=AT, spans=AT, groups=1, width=2)
    d.update(change)
    refused(lambda: va.kv_reorder(view(), **d), text)
    refused(lambda: va.kv_reorder(view(pos_stride=128), 1, 0, AT, AT, AT, 1, 2), "overlap")


def test_layouts_of_a_cache_taken_in_any_order():
    """Strides in any order are no overlap: refused only for what the host's memory is."""
    for kw in (dict(head_stride=64 * 128, pos_stride=128, seq_stride=2 * 64 * 128),
               dict(head_stride=128, seq_stride=256, pos_stride=3 * 256)):
        refused(lambda: va.kv_reorder(view(**kw), 2, 3 * 64 * 256, AT, AT, AT, 1, 2), "not device memory")
