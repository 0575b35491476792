"""The differential decode's scratch holds what can be split: at most two
results a range, whatever the number of requests."""
import pytest
import torch

from oracle import diff_ref

D, PAGE, BF = 128, 16, torch.bfloat16


@pytest.mark.parametrize("hq,hkv", [(64, 8), (64, 16), (32, 4), (16, 2)])
def test_scratch_does_not_grow_with_the_batch(tm, hq, hkv):
    size = tm._lib.load().tmopt_attn_decode_diff_workspace_size
    big, half = (size(b, hq, hkv, D, 0) for b in (8192, 4096))
    assert 0 < big - half <= 4096 * 4 + 256        # the page prefix alone
    # 512 ranges at most, two rows of 1 KB and an LSE per head and range
    assert big <= 2 * 512 * hq * 1028 + 8194 * 4 + 512
    assert size(8192, hq, hkv, D, 7) < big


@pytest.mark.gpu
@pytest.mark.parametrize("ends,hq,hkv,call", [
    ([700] * 300, 16, 2, {}), ([5000, 3, 0, 900], 32, 4, {}),
    ([50] * 30 + [3000], 64, 16, dict(num_workgroups=7)),
    ([90, 300] * 8, 8, 2, dict(min_pages=1)), ([2000], 24, 12, {}),
    ([170] * 65, 16, 4, dict(num_workgroups=64))])
def test_scratch_is_enough(tm, dev, ends, hq, hkv, call):
    """Exactly that many bytes, canaries on both sides."""
    g = torch.Generator().manual_seed(len(ends))
    rand = lambda *s: torch.randn(s, generator=g).to(BF).to(dev)   # noqa: E731
    pages = [-(-n // PAGE) for n in ends]
    table = torch.zeros((len(ends), max(pages)), dtype=torch.int32)
    perm, at = torch.randperm(sum(pages), generator=g).int(), 0
    for i, n in enumerate(pages):
        table[i, :n] = perm[at:at + n]
        at += n
    kp, vp = rand(at, PAGE, hkv, D), rand(at, PAGE, hkv, D)
    q, table = rand(len(ends), hq, D), table.to(dev)
    ctx = torch.tensor(ends, dtype=torch.int32, device=dev)
    lam = torch.full((hq // 2,), 0.6, device=dev)
    n = tm.decode_diff_workspace(len(ends), hq, hkv, dev,
                                 call.get("num_workgroups", 0)).numel()
    buf = torch.full((n + 8192,), 171, dtype=torch.uint8, device=dev)
    for _ in range(2):
        out, lse = tm.decode_diff_paged(q, kp, vp, table, ctx, lam, 0.1,
                                        workspace=buf[4096:4096 + n], **call)
        assert (buf[:4096] == 171).all() and (buf[4096 + n:] == 171).all()
        diff_ref.check(out, lse, diff_ref.decode(q, kp, vp, table, ctx, lam,
                                                 0.1))
