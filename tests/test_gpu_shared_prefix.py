"""PrefixBatch: slot maps, norm, rotation, cache and attention as one serving step.

Every step's outputs against a float64 computation that keeps each request's
keys and values in plain lists (rounded to the cache's type, as the cache
does). Tolerance 2e-2: a bf16 K or V may round the other way where the fp32
value lies on a tie, as everywhere in this engine.
"""

import pytest
import torch

from serving_reference import qk_norm_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,nh,nkv,hd", [(1, 4, 4, 64), (16, 8, 2, 128), (64, 6, 2, 64)])
def test_prefill_share_decode_roll_back_and_release(page, nh, nkv, hd):
    from loopspec_b200.shared_prefix import PrefixBatch
    R, prefix = 5, 150
    batch = PrefixBatch(1, nh, nkv, hd, n_blocks=-(-400 // page) + 40, page_size=page, max_requests=R, max_len=160,
                        max_tokens=200, max_positions=400)
    g = torch.Generator().manual_seed(page)
    qw, kw = (1 + 0.2 * torch.randn(2, hd, generator=g)).to(torch.bfloat16)
    rope = batch.rope.cpu()
    shared, own = [], [[] for _ in range(R)]

    def step(delta):
        new = [max(0, d) for d in delta]
        for i, d in enumerate(delta):
            del own[i][len(own[i]) + min(0, d):]
        n = sum(new)
        batch.begin(torch.tensor(delta, dtype=torch.int32, device="cuda"), n, max(new))
        if n == 0:
            return
        qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g).to(torch.bfloat16)
        pos = torch.tensor([len(shared) + len(own[i]) + j for i in range(R) for j in range(new[i])], dtype=torch.int32)
        q, k, v = qk_norm_reference(qkv, qw, kw, rope, pos, nh, nkv, hd, 1e-6, False)
        out = batch.attend(0, qkv.cuda(), qw.cuda(), kw.cuda()).double().cpu()
        t = 0
        for i in range(R):
            for _ in range(new[i]):
                own[i].append((k[t].to(torch.bfloat16).double(), v[t].to(torch.bfloat16).double()))
                keys, values = (torch.stack(x) for x in zip(*(shared + own[i])))
                rep = nh // nkv
                s = torch.einsum("hd,nhd->hn", q[t].to(torch.bfloat16).double(), keys.repeat_interleave(rep, 1)) / hd ** 0.5
                ref = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), values.repeat_interleave(rep, 1))
                assert float((out[t] - ref).abs().max()) < 2e-2
                t += 1

    step([0, 100, 0, 0, 0])
    step([0, prefix - 100, 0, 0, 0])
    batch.share(1, prefix)
    shared, own[1] = own[1], []
    step([7, 0, 33, 1, 150])
    step([1, 1, 1, 1, 1])
    step([4, 0, 4, 2, 4])
    step([-3, 0, -4, -1, -155])         # rejected drafts; the last request is released
    step([1, 1, 5, 0, 9])
    batch.check()
    assert batch.lens.tolist() == [len(x) for x in own]


def test_the_command_runs(capsys, monkeypatch):
    import sys

    from loopspec_b200 import shared_prefix
    monkeypatch.setattr(sys, "argv", ["shared_prefix", "--requests", "3", "--prefix", "70", "--prompt", "20", "--steps", "3",
                                      "--layers", "2", "--heads", "4", "--kv-heads", "2", "--dim", "64"])
    shared_prefix.main()
    assert "drafts" in capsys.readouterr().out
