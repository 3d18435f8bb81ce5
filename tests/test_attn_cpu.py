"""CPU tests of the attention entry points: the index functions their kernels reach memory through, and what the calls refuse
before anything is launched."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


@pytest.fixture(scope="module")
def lib():
    from tie_b200 import build, moe
    build.build_cuda()
    return moe.load_library()


def test_index_functions_stay_inside_whatever_a_step_says(tmp_path):
    from tie_b200 import build
    exe = tmp_path / "kv_index_check"
    subprocess.check_call([build._nvcc(), "-O2", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-o", str(exe),
                           os.path.join(ROOT, "tests", "kv_index_check.cu")])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout


FAKE = 1 << 20  # an address that is only looked at for its alignment: every call below is refused


def _cache(**kw):
    from tie_b200 import moe
    c = moe.KvCache.__new__(moe.KvCache)
    d = dict(type=moe.KV_F16, n_head_kv=4, head_dim=128, page_size=16, n_pages=8, k=FAKE, v=FAKE, k_scale=None, v_scale=None)
    for k, v in {**d, **kw}.items():
        setattr(c, k, v)
    return c


def _step(**kw):
    from tie_b200 import moe
    s = moe.KvStep.__new__(moe.KvStep)
    d = dict(n_seq=1, n_tokens=1, tok_start=FAKE, kv_len=FAKE, page_table=FAKE, max_pages=4, tree=None, pos=None)
    for k, v in {**d, **kw}.items():
        setattr(s, k, v)
    return s


def _attn(lib, cache, step, flags):
    return lib.tie_cuda_attn(None, ctypes.byref(cache), ctypes.byref(step), FAKE, 32, 1.0, FAKE, flags)


@pytest.mark.parametrize("what, code", [
    (dict(type=0), "ENOTSUP"), (dict(type=4), "ENOTSUP"), (dict(head_dim=96), "ENOTSUP"), (dict(head_dim=256), "ENOTSUP"),
    (dict(n_head_kv=0), "EINVAL"), (dict(n_head_kv=257), "EINVAL"), (dict(page_size=8), "EINVAL"), (dict(page_size=48), "EINVAL"),
    (dict(page_size=1 << 17), "EINVAL"), (dict(n_pages=0), "EINVAL"), (dict(k=None), "EINVAL"), (dict(v=FAKE + 8), "EINVAL"),
    (dict(type=3), "EINVAL"), (dict(type=3, k_scale=FAKE, v_scale=FAKE + 2), "EINVAL"),
])
def test_caches_that_are_refused(lib, what, code):
    from tie_b200 import moe
    assert _attn(lib, _cache(**what), _step(), moe.DEVICE) == getattr(moe, code)


@pytest.mark.parametrize("what", [
    dict(n_seq=0), dict(n_seq=1025), dict(n_tokens=-1), dict(tok_start=None), dict(kv_len=None), dict(page_table=None),
    dict(max_pages=0), dict(max_pages=1 << 27), dict(n_tokens=1 << 30), dict(n_tokens=1 << 26), dict(tok_start=FAKE + 2), dict(pos=FAKE + 1), dict(tree=FAKE + 4),
])
def test_steps_that_are_refused(lib, what):
    from tie_b200 import moe
    assert _attn(lib, _cache(), _step(**what), moe.DEVICE) == moe.EINVAL


def test_no_context_host_pointers_and_null_descriptions_are_refused(lib):
    from tie_b200 import moe
    cache, step = _cache(), _step()
    assert _attn(lib, cache, step, moe.DEVICE) == moe.EINVAL  # no context
    assert _attn(lib, cache, step, moe.HOST) == moe.EINVAL
    assert lib.tie_cuda_attn(None, None, ctypes.byref(step), FAKE, 32, 1.0, FAKE, moe.DEVICE) == moe.EINVAL
    assert lib.tie_cuda_kv_read(None, ctypes.byref(cache), None, FAKE, FAKE, 0, moe.DEVICE) == moe.EINVAL
    assert lib.tie_cuda_qk_norm_rope(None, ctypes.byref(cache), ctypes.byref(step), None, moe.DEVICE) == moe.EINVAL


def test_descriptions_have_the_layout_of_the_header(tmp_path):
    """Field offsets of the ctypes structures against the header's, as a C compiler sees them."""
    from tie_b200 import moe
    pairs = [("tie_cuda_kv_cache", moe.KvCache), ("tie_cuda_kv_step", moe.KvStep), ("tie_cuda_attn_qkv", moe.AttnQkv),
             ("tie_cuda_attn_weights", moe.AttnWeights)]
    body = "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for n, t in pairs for f, _ in t._fields_)
    body += "".join(f'printf("%zu\\n", sizeof({n}));' for n, _ in pairs)
    src = tmp_path / "o.c"
    src.write_text(f'#include <stdio.h>\n#include "tie_cuda.h"\nint main(void){{ {body} return 0; }}\n')
    exe = tmp_path / "o"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    want = [getattr(t, f).offset for _, t in pairs for f, _ in t._fields_] + [ctypes.sizeof(t) for _, t in pairs]
    assert [int(x) for x in subprocess.check_output([str(exe)], text=True).split()] == want
