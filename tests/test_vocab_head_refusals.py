"""What the vocabulary-head operators refuse, without a GPU: the argument checks come before any launch."""
import ctypes
import math

import pytest
import torch

BF16 = torch.bfloat16


def args(T=4, H=64, V=10, dtype=BF16):
    return torch.zeros(T, H, dtype=dtype), torch.zeros(V, H, dtype=dtype), torch.zeros(T, dtype=torch.int64)


def test_cpu_tensors_are_refused_not_computed_elsewhere():
    from spatialthinker_amd import ops
    from verl.utils import torch_functional as VF
    h, w, lab = args()
    with pytest.raises(RuntimeError, match="not on a GPU"):
        ops.linear_logprob_fwd(h, w, lab)
    with pytest.raises(RuntimeError, match="not on a GPU"):
        VF.linear_log_probs(h, w, lab)
    with pytest.raises(RuntimeError, match="not on a GPU"):
        VF.linear_topk_kl(h, w, torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="not on a GPU"):
        VF.top_log_probs(torch.zeros(2, 50), 3)


@pytest.mark.parametrize("temperature", [0.0, -1.0, math.inf, math.nan, 1e-320, 1e-38, 1e38])
def test_temperature(temperature):
    from spatialthinker_amd import ops
    h, w, lab = args()
    with pytest.raises(ValueError, match="temperature"):
        ops.linear_logprob_fwd(h, w, lab, temperature)
    with pytest.raises(ValueError, match="temperature"):
        ops.topk_logprob(w, 3, temperature)


def test_types_and_shapes():
    from spatialthinker_amd import ops
    from verl.utils import torch_functional as VF
    h, w, lab = args()
    with pytest.raises(TypeError):
        ops.linear_logprob_fwd(h.float(), w, lab)
    with pytest.raises(TypeError):
        ops.linear_logprob_fwd(h, w.half(), lab)
    with pytest.raises(ValueError):
        ops.linear_logprob_fwd(*args(H=72)[:2], lab)               # width not a multiple of 64
    with pytest.raises(ValueError):
        ops.linear_logprob_fwd(h, torch.zeros(10, 128, dtype=BF16), lab)
    with pytest.raises(ValueError):
        ops.linear_logprob_fwd(h, torch.zeros(0, 64, dtype=BF16), lab)
    with pytest.raises(ValueError):                                # rows that are not 16-byte aligned
        ops.linear_logprob_fwd(torch.zeros(4, 65, dtype=BF16)[:, :64], w, lab)
    with pytest.raises(ValueError):
        ops.linear_logprob_fwd(torch.zeros(1, 64, dtype=BF16).expand(4, 64), w, lab)       # rows that overlap
    with pytest.raises(ValueError):
        VF.linear_log_probs(h, w, lab[:3])
    with pytest.raises(ValueError):
        VF.linear_topk_kl(h, w, torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 2))
    with pytest.raises(ValueError):
        VF.linear_topk_kl(h, w, torch.zeros(5, 3, dtype=torch.int32), torch.zeros(5, 3))
    for k in (0, 11, -1):
        with pytest.raises(ValueError):
            ops.topk_logprob(torch.zeros(2, 10, dtype=BF16), k)
    with pytest.raises(ValueError):
        ops.topk_logprob(torch.zeros(2, 1000, dtype=BF16), 257)
    with pytest.raises(TypeError):
        ops.topk_logprob(torch.zeros(2, 1000), 2)
    with pytest.raises(ValueError):
        ops.topk_logprob(torch.zeros(1, 1000, dtype=BF16).expand(2, 1000), 2)


def test_c_entries_return_einval_before_any_launch():
    from spatialthinker_amd.lib import lib
    L = lib()
    n = ctypes.c_int64(0)
    at = ctypes.addressof(n)
    assert L.st_linear_head_workspace_bytes.raw(8, 1000, 64, 4, 1, at, None) == 0 and n.value > 0
    small = n.value
    assert L.st_linear_head_workspace_bytes.raw(8, 1000, 64, 4, 0, at, None) == 0 and n.value > 0
    for T, V, H, K in ((-1, 10, 64, 0), (8, 0, 64, 0), (8, 10, 0, 0), (8, 10, 65, 0), (8, 10, 64, 1025), (8, 10, 64, -1), (8, (1 << 21) + 1, 64, 0)):
        assert L.st_linear_head_workspace_bytes.raw(T, V, H, K, 1, at, None) == -22
    p = 1 << 20                                                    # never touched: every call below is refused
    fwd = lambda h=p, ldh=64, w=p, ldw=64, lab=p, it=1.0, ws=p, nb=1 << 40, T=8, V=1000, H=64, z=None, ldz=0: L.st_linear_logprob_fwd.raw(
        h, ldh, w, ldw, lab, it, p, p, z, ldz, ws, nb, T, V, H, None)
    for bad in (dict(h=None), dict(w=None), dict(lab=None), dict(ldh=63), dict(ldw=68), dict(ldh=56), dict(ldw=1 << 22), dict(h=p + 2), dict(w=p + 8),
                dict(it=0.0), dict(it=-1.0), dict(it=math.inf), dict(it=math.nan), dict(ws=None), dict(nb=small // 1000), dict(T=-1), dict(V=0), dict(H=65),
                dict(z=p + 4, ldz=1024), dict(z=p, ldz=1023), dict(z=p, ldz=1022), dict(z=p, ldz=1020)):
        assert fwd(**bad) == -22, bad
    bwd = lambda dh=p, lddh=64, db=None, df=None, lddw=64, acc=0, ws=p, nb=1 << 40, z=None, ldz=0: L.st_linear_logprob_bwd.raw(
        p, 64, p, 64, p, p, p, p, 1.0, z, ldz, dh, lddh, db, df, lddw, acc, ws, nb, 8, 1000, 64, None)
    for bad in (dict(dh=p + 2), dict(lddh=63), dict(lddh=60), dict(db=p, df=p), dict(db=p, acc=1), dict(db=p, lddw=66), dict(df=p, lddw=62), dict(df=p + 4),
                dict(ws=None), dict(nb=small - 1), dict(z=p + 8, ldz=1024), dict(z=p, ldz=1000)):
        assert bwd(**bad) == -22, bad
    kl = lambda K=4, ids=p, a=p, ws=p, T=8: L.st_linear_topk_kl_fwd.raw(p, 64, p, 64, ids, a, K, 0, 1.0, p, p, p, None, 0, ws, 1 << 40, T, 1000, 64, None)
    for bad in (dict(K=0), dict(K=1025), dict(ids=None), dict(a=None), dict(ws=None), dict(K=1024, T=1 << 21)):
        assert kl(**bad) == -22, bad
    top = lambda z=p, ldl=1000, k=5, it=1.0, ws=p, nb=1 << 40, T=8, V=1000: L.st_topk_logprob.raw(z, ldl, k, it, p, p, p, ws, nb, T, V, None)
    for bad in (dict(z=None), dict(z=p + 1), dict(ldl=999), dict(k=0), dict(k=257), dict(k=6, V=5, ldl=5), dict(it=0.0), dict(T=-1), dict(V=0)):
        assert top(**bad) == -22, bad


def test_kept_logits_buffers():
    from spatialthinker_amd import ops
    h, w, lab = args(T=4, V=70)
    good = ops.head_logits_buffer(4, 70, h.device)
    assert good.shape == (4, 128) and good.dtype == torch.float32
    for bad in (good.double(), good.to(BF16)):
        with pytest.raises(TypeError):
            ops._kept_logits(bad, 4, 70, h.device)
    for bad in (good[:3], good[:, :64], good[0], good[:1].expand(4, 128), torch.zeros(4, 130)[:, :128], torch.zeros(4, 132)[:, 1:129]):
        with pytest.raises(ValueError):
            ops._kept_logits(bad, 4, 70, h.device)
    assert ops._kept_logits(None, 4, 70, h.device) == (None, 0) and ops._kept_logits(torch.zeros(4, 132)[:, :128], 4, 70, h.device)[1] == 132


def test_rows_at_any_pitch_reach_the_kernels():
    """The last position of each sequence, whose rows lie a whole sequence apart (here 2^22 elements, more than the kernels address): copied, not refused.
    What is refused here is only the CPU tensor behind it."""
    from verl.utils import torch_functional as VF
    last = torch.zeros(2, 2048, 2048, dtype=BF16)[:, -1]
    assert last.stride(0) == 1 << 22
    with pytest.raises(RuntimeError, match="not on a GPU"):
        VF.linear_log_probs(last, torch.zeros(10, 2048, dtype=BF16), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="not on a GPU"):
        VF.linear_log_probs(torch.zeros(2, 2048, dtype=BF16), torch.zeros(2, 2048, 2048, dtype=BF16)[:, -1], torch.zeros(2, dtype=torch.int64))
    near = torch.zeros(2, 2048, 2048 - 8, dtype=BF16)[:, -1]
    assert VF._rows16(near) is near                                # a pitch below it is used as it lies


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_teacher_ids_of_every_integer_type(dtype):
    from verl.utils import torch_functional as VF
    h, w, _ = args()
    with pytest.raises(RuntimeError, match="not on a GPU"):
        VF.linear_topk_kl(h, w, torch.ones(4, 3, dtype=dtype), torch.zeros(4, 3))


def test_no_teacher_entries_at_all_is_an_argument_error():
    from verl.utils import torch_functional as VF
    h, w, _ = args()
    with pytest.raises(ValueError, match="ids"):
        VF.linear_topk_kl(h, w, torch.zeros(4, 0, dtype=torch.int32), torch.zeros(4, 0))


def test_top_log_probs_of_overlapping_rows_and_single_columns():
    """Expanded logits and a vocabulary of one token in any layout are copied; the kernel entry itself goes on refusing them."""
    from spatialthinker_amd import ops
    from verl.utils import torch_functional as VF
    shared = torch.zeros(1, 50, dtype=BF16).expand(3, 50)
    column = torch.zeros(3, 4, dtype=BF16)[:, 1:2].t().contiguous().t()
    assert column.stride(-1) != 1
    for z, k in ((shared, 3), (column, 1), (torch.zeros(40, dtype=BF16).as_strided((3, 20), (4, 1)), 2)):
        with pytest.raises(ValueError):
            ops.topk_logprob(z, k)
        with pytest.raises(RuntimeError, match="not on a GPU"):
            VF.top_log_probs(z, k)


def test_workspace_is_what_the_rows_need():
    """d of a piece takes at most 512 MiB or, beyond 2^20 rows, 256 columns per row, and never more columns than the vocabulary has; the partial sums of dh
    one fp32 T x H and at most 512 MiB more."""
    from spatialthinker_amd.lib import lib
    n = ctypes.c_int64(0)

    def need(T, V, H):
        assert lib().st_linear_head_workspace_bytes.raw(T, V, H, 0, 1, ctypes.addressof(n), None) == 0
        return n.value
    up = lambda x, a: (x + a - 1) // a * a
    for T in (1, 64, 65, 128, 129, 256, 257, 1000, 4096, 8192, 65536, 1 << 20, 65535 * 64 + 100):
        for V in (1, 5, 64, 65, 300, 32513, 152064, 1 << 21):
            for H in (64, 2048, 8192):
                rows = up(T, 64)
                d = min(max(512 << 20, rows * 512), rows * up(V, 64) * 2)
                fixed = 20 * T + rows * H * 2 + T * H * 4 + (2 if T <= 128 else 1) * d
                slabs = need(T, V, H) - fixed
                assert slabs <= (512 << 20) + 256 * 8, (T, V, H, slabs)
    few = need(65535 * 64 + 100, 5, 64)
    assert few <= (65535 * 64 + 100) * (20 + 128 + 256 + 128) + 64 * 300 + 256 * 8    # 64 columns of d, not a tile's 256


def test_workspaces_that_are_not_aligned_are_refused():
    """The kernels store 16 bytes at a time into the workspace."""
    from spatialthinker_amd.lib import lib
    L, p = lib(), 1 << 20                                          # never touched: every call below is refused
    for off in (1, 4, 8):
        ws = p + off
        assert L.st_linear_logprob_fwd.raw(p, 64, p, 64, p, 1.0, p, p, None, 0, ws, 1 << 40, 8, 1000, 64, None) == -22
        assert L.st_linear_logprob_bwd.raw(p, 64, p, 64, p, p, p, p, 1.0, None, 0, p, 64, None, None, 0, 0, ws, 1 << 40, 8, 1000, 64, None) == -22
        assert L.st_linear_topk_kl_fwd.raw(p, 64, p, 64, p, p, 4, 0, 1.0, p, p, p, None, 0, ws, 1 << 40, 8, 1000, 64, None) == -22
        assert L.st_linear_topk_kl_bwd.raw(p, 64, p, 64, p, p, 4, 0, 1.0, p, p, p, None, 0, p, 64, None, None, 0, 0, ws, 1 << 40, 8, 1000, 64, None) == -22
