"""CPU: the answering end's library exports what include/toktier_head.h
declares, checks its arguments before it touches a device, and the 8-bit
format of ``quantize_fp8`` is the one the header describes."""

from __future__ import annotations

import ctypes as C
import math
import re
from pathlib import Path

import pytest
import torch

from toktier_amd import head

HEADER = Path(__file__).resolve().parent.parent / "include" / "toktier_head.h"


def test_header_and_library_agree():
    text = HEADER.read_text()
    names = set(re.findall(r"\b(tk_head_[a-z_]+)\s*\(", text.split("extern \"C\"")[1]))
    assert names == set(head.SYMBOLS)
    for name in names:
        assert hasattr(head.lib(), name), name
    defines = dict(re.findall(r"#define\s+(TKH_[A-Z0-9_]+)\s+(\d+)\b", text))
    assert [int(defines[n]) for n in ("TKH_F32", "TKH_BF16", "TKH_F16")] == [
        head.TKH_F32, head.TKH_BF16, head.TKH_F16]
    from toktier_amd import _ffi
    codes = re.findall(r"#define\s+TKH_(E_[A-Z_]+)\s+\((-\d+)\)", text)
    assert codes and all(getattr(_ffi, "TK_" + n) == int(v) for n, v in codes)


def test_packed_arguments_have_the_structs_layout():
    """The format strings against the header's fields, in order."""
    kind = {"int64_t": "q", "uint64_t": "Q", "int32_t": "i", "float": "f"}
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name, packed in (("tkh_norm", head._NORM), ("tkh_matmul", head._MATMUL),
                         ("tkh_sample", head._SAMPLE)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        want = ""
        for line in body.split(";"):
            line = line.strip()
            if line:
                first = re.sub(r"^const\s+", "", line)
                want += "Q" if "*" in line else kind[first.split()[0]] * (line.count(",") + 1)
        flat = re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), packed.format)
        assert flat == want, name


def call(name, packed, *values):
    return getattr(head.lib(), name)(packed.pack(*values), None)


def message() -> str:
    return head.lib().tk_head_last_error().decode()


def test_refusals_without_a_device():
    L = head.lib()
    for name in ("tk_head_norm", "tk_head_matmul", "tk_head_sample"):
        assert getattr(L, name)(None, None) == -1
    p = 1 << 20  # an address that no call reads
    norm = [p, 0, p, p, p, 0, 4, 256, 256, 0, 256, 2, 0, 1e-6, 0, 0, 0]

    def refused(name, packed, args, at, value, status, word):
        args = list(args)
        args[at] = value
        assert call(name, packed, *args) == status, (name, at, value)
        assert word in message(), message()

    for at, value, status, word in (
            (0, 0, -1, "null"), (7, 0, -2, "k 0"), (7, 65537, -9, "65537"), (6, -1, -2, "rows -1"),
            (10, 200, -2, "16-byte"), (10, 248, -2, "16-byte"), (3, p + 4, -2, "16-byte"),
            (11, 1, -2, "scale"), (14, 3, -9, "dtype"), (15, 1, -9, "weight"), (8, -8, -2, "stride")):
        refused("tk_head_norm", head._NORM, norm, at, value, status, word)
    mm = [p, p, p, p, p, 4, 64, 256, 256, 2, 256, 2, 64, 1, 0]
    for at, value, status, word in (
            (2, 0, -1, "null"), (7, 0, -2, "k 0"), (8, 264, -2, "16-byte"), (0, p + 8, -2, "16-byte"),
            (8, 240, -2, "stride"), (11, 1, -2, "stride"), (12, 63, -2, "stride"),
            (13, 9, -9, "dtype"), (13, 0, -9, "dtype"), (6, 1 << 40, -2, "n ")):
        refused("tk_head_matmul", head._MATMUL, mm, at, value, status, word)
    sm = [p, p, 0, 0, 0, 0, 0, p, 0, p, 1 << 40, 4, 1000, 1000, 0, 1.0, 0, 1.0, 0.0, 0, 0]
    for at, value, status, word in (
            (0, 0, -1, "null"), (12, 0, -2, "vocab 0"), (12, 1 << 25, -2, "vocab"),
            (19, 5, -9, "dtype"), (13, -1, -2, "stride")):
        refused("tk_head_sample", head._SAMPLE, sm, at, value, status, word)
    sm[6], sm[14] = p, 31
    assert call("tk_head_sample", head._SAMPLE, *sm) == -2 and "32 words" in message()


def test_a_vocabulary_ends_where_masses_would_pass_64_bits():
    """2**24 equal logits would weigh 2**64."""
    p = 1 << 20  # an address that no call reads
    values = [p, p, 0, 0, 0, 0, 0, p, 0, p, 1 << 62, 4, 1 << 24, 1 << 24, 0, 1.0, 0, 1.0, 0.0, 0, 0]
    assert call("tk_head_sample", head._SAMPLE, *values) == -2
    assert "vocab" in message()
    size = head.lib().tk_head_sample_workspace
    assert size(4, 1 << 24, 0) == 0 and size(4, (1 << 24) - 1, 0) > 0


def test_sizes_that_no_launch_holds_are_refused():
    """A launch has fewer than 2**32 threads along an axis: a norm's row of 256
    values takes 64, one of 65536 values 1024, a sampled row 1024, 64 rows of
    weights 256, four runs of 1024 logits 256."""
    p = 1 << 20  # an address that no call reads

    def norm(rows, k):
        return call("tk_head_norm", head._NORM, p, 0, p, p, p, 0, rows, k, k, 0, k, k // 128, 0, 1e-6, 0, 0, 0)

    def matmul(m, n):
        return call("tk_head_matmul", head._MATMUL, p, p, p, p, p, m, n, 256, 256, 2, 256, 2, n, 1, 0)

    def sample(rows, vocab):
        return call("tk_head_sample", head._SAMPLE, p, p, 0, 0, 0, 0, 0, p, 0, p, 1 << 62, rows, vocab, vocab, 0,
                    1.0, 0, 1.0, 0.0, 0, 0)

    for refused, args, words in ((norm, (1 << 26, 256), ("rows 67108864",)),
                                 (norm, (1 << 22, 65536), ("rows 4194304",)),
                                 (matmul, (1, 1 << 30), ("n 1073741824",)),
                                 (matmul, (1_000_000, 1 << 20), ("m 1000000",)),
                                 (sample, (1 << 22, 100), ("rows 4194304",)),
                                 (sample, (1 << 12, (1 << 24) - 1), ("rows 4096", "vocab 16777215"))):
        assert refused(*args) == -2 and all(w in message() for w in words), message()


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is visible")
def test_the_largest_sizes_pass_the_checks():
    """As above, one less: refused for the missing device alone."""
    p = 1 << 20
    for rows, k in (((1 << 26) - 1, 256), ((1 << 22) - 1, 65536)):
        assert call("tk_head_norm", head._NORM, p, 0, p, p, p, 0, rows, k, k, 0, k, k // 128, 0, 1e-6, 0, 0, 0) == -3
    n = (1 << 30) - 64
    assert call("tk_head_matmul", head._MATMUL, p, p, p, p, p, 1, n, 256, 256, 2, 256, 2, n, 1, 0) == -3
    for rows, vocab in (((1 << 22) - 1, 100), ((1 << 12) - 1, (1 << 24) - 1)):
        assert call("tk_head_sample", head._SAMPLE, p, p, 0, 0, 0, 0, 0, p, 0, p, 1 << 62, rows, vocab, vocab, 0,
                    1.0, 0, 1.0, 0.0, 0, 0) == -3


def test_nothing_to_do_needs_no_device():
    assert call("tk_head_norm", head._NORM, 0, 0, 0, 0, 0, 0, 0, 256, 0, 0, 256, 2, 0, 1e-6, 0, 0, 0) == 0
    assert call("tk_head_matmul", head._MATMUL, 0, 0, 0, 0, 0, 0, 64, 256, 256, 2, 256, 2, 64, 1, 0) == 0
    assert call("tk_head_sample", head._SAMPLE, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1000, 1000, 0,
                1.0, 0, 1.0, 0.0, 0, 0) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is visible")
def test_calls_without_a_device_fail():
    p = 1 << 20
    status = call("tk_head_norm", head._NORM, p, 0, p, p, p, 0, 4, 256, 256, 0, 256, 2, 0, 1e-6, 0, 0, 0)
    assert status == -3 and message()
    with pytest.raises(ValueError, match="GPU"):
        head.rms_norm_fp8(torch.zeros(2, 4), torch.zeros(4))
    with pytest.raises(ValueError, match="GPU"):
        head.sample(torch.zeros(2, 4), torch.zeros(2))


@pytest.mark.parametrize("k", [1, 100, 128, 300])
def test_quantize_format(k):
    g = torch.Generator().manual_seed(k)
    x = torch.randn(9, k, generator=g) * torch.exp(4 * torch.randn(9, 1, generator=g))
    x[3] = 0.0
    q, s = head.quantize_fp8(x, chunk=4)
    assert q.shape == (9, k) and q.stride(0) % 128 == 0 and q.data_ptr() % 16 == 0
    e = s.view(torch.uint8).long() - 127
    scale = torch.exp2(e.double()).repeat_interleave(128, 1)[:, :k]
    back = q.float().double() * scale
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)
    assert bool(((back - x.double()).abs() <= bound).all())
    blocks = torch.nn.functional.pad(x, (0, -k % 128)).unflatten(1, (-1, 128)).abs().amax(-1).double()
    unit = torch.exp2(e.double())
    assert bool((blocks <= 448 * unit).all())
    assert bool(((blocks > 224 * unit) | ((blocks == 0) & (e == 0))).all())


def test_quantize_edges():
    x = torch.zeros(1, 256)
    x[0, 0], x[0, 128], x[0, 129] = 448.0, 448.00003, math.inf
    q, s = head.quantize_fp8(x)
    assert s.view(torch.uint8).tolist() == [[127, 128]]
    assert float(q[0, 0].float()) == 448 and bool(q[0, 129].float().isnan())
    with pytest.raises(ValueError):
        head.quantize_fp8(torch.zeros(4))
    with pytest.raises(ValueError):
        head.OutputHead(torch.ones(256), q, s, vocab=2)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is visible")
def test_strides_of_a_single_row_are_not_asked_about():
    """No kernel steps from one row to the next where there is one: refused
    for the missing device alone."""
    p = 1 << 20
    mm = [p, p, p, p, p, 1, 64, 1000, 1000, 8, 1008, 8, 64, 1, 0]
    assert call("tk_head_matmul", head._MATMUL, *mm) == -3
    mm = [p, p, p, p, p, 4, 1, 1000, 1008, 8, 1000, 8, 1, 1, 0]
    assert call("tk_head_matmul", head._MATMUL, *mm) == -3
    norm = [p, p, p, p, p, p, 1, 256, -8, -8, 256, 2, -8, 1e-6, 0, 0, 0]
    assert call("tk_head_norm", head._NORM, *norm) == -3


class Stand:
    """What the Python side calls: notes it and queues nothing."""

    def __init__(self):
        self.calls = []

    def tk_head_norm(self, args, stream):
        self.calls.append(("norm", head._NORM.unpack(args)))
        return 0

    def tk_head_matmul(self, args, stream):
        self.calls.append(("matmul", head._MATMUL.unpack(args)))
        return 0

    def tk_head_sample(self, args, stream):
        self.calls.append(("sample", head._SAMPLE.unpack(args)))
        return 0

    def tk_head_sample_workspace(self, rows, vocab, dtype):
        return 64

    def names(self):
        return [name for name, _ in self.calls]


class Place:
    index = 0


@pytest.fixture
def stand(monkeypatch):
    """The checks of ``toktier_amd.head`` on CPU tensors."""
    s = Stand()
    monkeypatch.setattr(head, "_lib", s)
    monkeypatch.setattr(head, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(head, "_gpu", lambda t, name: Place)
    monkeypatch.setattr(head, "_on", lambda t, device, name: None)
    return s


def test_a_weight_of_one_value_is_dense(stand):
    head.rms_norm_fp8(torch.randn(3, 1), torch.randn(1, 5)[:, 0])
    assert stand.names() == ["norm"]
    with pytest.raises(ValueError, match="dense"):
        head.rms_norm_fp8(torch.randn(3, 2), torch.randn(2, 5)[:, 0])


def eight(*shape):
    return head.quantize_fp8(torch.randn(*shape))


@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (0,), (0, 3), (3, 0), (1, 1, 1)])
@pytest.mark.parametrize("k", [256, 300])
def test_any_number_of_leading_axes(stand, lead, k):
    blocks = (k + 127) // 128
    x, w = torch.randn(*lead, k), torch.ones(k)
    r = torch.randn(*lead, k)
    out = head.rms_norm_fp8(x, w, residual=r, residual_out=r)
    assert out.q.shape == lead + (k,) and out.scale.shape == lead + (blocks,)
    assert out.residual is r
    assert head.rms_norm_fp8(x, w, residual=r).residual.shape == x.shape
    for n in (40, 41):
        assert head.matmul_fp8(out.q, out.scale, *eight(n, k)).shape == lead + (n,)
        given = torch.empty(*lead, n, dtype=torch.bfloat16)
        assert head.matmul_fp8(out.q, out.scale, *eight(n, k), out=given) is given
        assert head.OutputHead(w, *eight(n, k)).logits(x, residual=r).shape == lead + (n,)
    # what the kernels are given lies in what comes back
    args = stand.calls[0][1]
    assert args[3] == out.q.data_ptr() and args[4] == out.scale.data_ptr() and args[5] == r.data_ptr()


def test_next_ids_of_other_than_rows_queues_nothing(stand):
    out = head.OutputHead(torch.ones(256), *eight(40, 256))
    for shape in ((256,), (1, 1, 256)):
        with pytest.raises(ValueError, match="two axes"):
            out.next_ids(torch.randn(*shape), torch.rand(1))
    assert stand.names() == []


def needs(t):
    return t.requires_grad_(True)


def test_outputs_of_inputs_that_require_grad_have_no_backward(stand):
    x, w, r = torch.randn(2, 256), torch.ones(256), torch.randn(2, 256)
    plain = head.rms_norm_fp8(x, w, residual=r)
    assert not any(t.requires_grad for t in plain)
    for kw in (dict(x=needs(x.clone()), weight=w), dict(x=x, weight=needs(w.clone())),
               dict(x=x, weight=w, residual=needs(r.clone())),
               dict(x=needs(x.clone()), weight=w, residual=r)):
        out = head.rms_norm_fp8(**kw)
        assert (out.residual is None) == ("residual" not in kw)
        for t in out:
            if t is not None:
                with pytest.raises(NotImplementedError, match="rms_norm_fp8"):
                    t.float().sum().backward()
        with torch.no_grad():
            assert not any(t.requires_grad for t in head.rms_norm_fp8(**kw) if t is not None)
    # the sum does not depend on the weight
    out = head.rms_norm_fp8(x, needs(w.clone()), residual=r, residual_out=r)
    assert out.residual is r and not r.requires_grad and out.q.requires_grad

    a, b = eight(2, 256), eight(40, 256)
    assert not head.matmul_fp8(*a, *b).requires_grad
    for n in (40, 41):
        c = head.matmul_fp8(out.q, out.scale, *eight(n, 256))
        with pytest.raises(NotImplementedError, match="matmul_fp8"):
            c.float().sum().backward()
    logits, u = torch.randn(2, 40), torch.rand(2)
    t = torch.ones(2)
    assert not head.sample(logits, u, temperature=t).logprob.requires_grad
    for kw in (dict(logits=needs(logits.clone())), dict(logits=logits, temperature=needs(t.clone()))):
        got = head.sample(u=u, **kw)
        assert not got.ids.requires_grad
        with pytest.raises(NotImplementedError, match="sample"):
            got.logprob.sum().backward()


def test_nothing_that_requires_grad_is_written_into_a_given_tensor(stand):
    x, w, r = torch.randn(2, 256), torch.ones(256), torch.randn(2, 256)
    a, b, out = eight(2, 256), eight(40, 256), torch.empty(2, 40, dtype=torch.bfloat16)
    grad = needs(r.clone())
    for kw in (dict(x=needs(x.clone()), weight=w, residual=r, residual_out=r),
               dict(x=x, weight=w, residual=grad, residual_out=torch.empty_like(r)),
               dict(x=x, weight=w, residual=r, residual_out=grad)):
        with pytest.raises(ValueError, match="residual_out"):
            head.rms_norm_fp8(**kw)
    with pytest.raises(ValueError, match="out"):
        head.matmul_fp8(needs(a[0].clone()), a[1], *b, out=out)
    with pytest.raises(ValueError, match="out"):
        head.matmul_fp8(*a, *b, out=needs(out.clone()))
    assert stand.names() == []
    with torch.no_grad():
        assert head.rms_norm_fp8(x, w, residual=grad, residual_out=grad).residual is grad


def test_an_output_head_holds_its_weights_detached(stand):
    w = torch.nn.Parameter(torch.ones(256))
    out = head.OutputHead(w, *head.quantize_fp8(torch.nn.Parameter(torch.randn(40, 256))))
    assert out.norm_weight.data_ptr() == w.data_ptr()
    assert not out.logits(torch.randn(2, 256)).requires_grad
    got = out.next_ids(needs(torch.randn(2, 256)), torch.rand(2))
    with pytest.raises(NotImplementedError):
        got.logprob.sum().backward()


def test_what_is_written_in_place_is_known_to_autograd(stand):
    """A graph that saved a tensor notices that a call wrote over it."""
    x, w, r = torch.randn(2, 256), torch.ones(256), torch.randn(2, 256)
    a, b, out = eight(2, 256), eight(40, 256), torch.zeros(2, 40, dtype=torch.bfloat16)
    read = [(t, t._version) for t in (x, w, *a, *b)]
    factor = needs(torch.ones(2, 256))
    saved = (factor * r).sum()
    head.rms_norm_fp8(x, w, residual=r, residual_out=r)
    with pytest.raises(RuntimeError, match="inplace"):
        saved.backward()
    saved = (needs(torch.ones(2, 40, dtype=torch.bfloat16)) * out).sum()
    head.matmul_fp8(*a, *b, out=out)
    with pytest.raises(RuntimeError, match="inplace"):
        saved.backward()
    # what is only read is not marked
    assert all(t._version == version for t, version in read)
    with torch.inference_mode():
        kept = torch.randn(2, 256)
        assert head.rms_norm_fp8(kept, w, residual=kept, residual_out=kept).residual is kept


def test_the_librarys_arguments_are_those_that_are_packed():
    defined = int(re.search(r"#define\s+TKH_ABI_VERSION\s+(\d+)", HEADER.read_text()).group(1))
    assert head.lib().tk_head_abi_version() == head.ABI_VERSION == defined
    # csrc/head/head_api.cpp holds the structs to the same sizes
    assert (head._NORM.size, head._MATMUL.size, head._SAMPLE.size) == (120, 112, 144)


def test_a_library_of_other_arguments_is_refused(tmp_path):
    import subprocess
    names = [n for n in head.SYMBOLS if n != "tk_head_abi_version"]
    for extra in ("", "int tk_head_abi_version(void) { return %d; }" % (head.ABI_VERSION + 1)):
        src, so = tmp_path / "other.c", tmp_path / f"other{len(extra)}.so"
        src.write_text("".join(f"int {n}(void) {{ return 0; }}\n" for n in names) + extra)
        subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
        with pytest.raises(RuntimeError, match="build it again"):
            head.lib(so)


def test_the_library_is_of_the_present_sources(monkeypatch, tmp_path):
    from toktier_amd import _build
    assert _build.verify_head() is None
    here = tmp_path / "head"
    here.mkdir()
    for f in _build.HEAD_SRC.iterdir():
        (here / f.name).write_bytes(f.read_bytes())
    monkeypatch.setattr(_build, "HEAD_SRC", here)
    assert _build.verify_head() is None
    with open(here / "head_common.h", "a") as f:
        f.write("// edited\n")
    assert "sources" in _build.verify_head()
    with pytest.warns(RuntimeWarning, match="sources"):
        head.lib(_build.HEAD_LIB)
    monkeypatch.setattr(_build, "HEAD_LIB", tmp_path / "none.so")
    assert "missing" in _build.verify_head()


def test_settings_of_another_kind_are_type_errors(stand):
    logits, u = torch.randn(2, 40), torch.rand(2)
    for kw in (dict(top_k=5.0), dict(top_k="5"), dict(temperature="1"), dict(top_p=None), dict(min_p=[0.1])):
        with pytest.raises(TypeError, match=next(iter(kw))):
            head.sample(logits, u, **kw)
    for eps in ("1e-6", None):
        with pytest.raises(TypeError, match="eps"):
            head.rms_norm_fp8(torch.randn(2, 40), torch.ones(40), eps=eps)
    assert stand.names() == []
    import numpy as np
    head.sample(logits, u, top_k=np.int64(5), temperature=np.float32(0.5), top_p=1)
    assert stand.calls[-1][1][16] == 5 and stand.calls[-1][1][15] == 0.5
