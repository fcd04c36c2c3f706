"""More cases of the likelihood and distillation tests, run on the device they are given."""

import torch

import cherimoya_b200 as cb
import likelihood_common as C


def case_candidates(dev, dtype, v, rows):
    """Rows in which a block finds more candidates for its top entries than it ranks and has
    room for all of them: equal ones, ones that share their 16-byte vectors, and more than
    there is room for, in neighbouring rows, so that one launch takes each way."""
    g = torch.Generator().manual_seed(v + rows)
    z = -1.0 - torch.rand(rows, v, generator=g)
    for r in range(rows):
        at = torch.randperm(v // 8 - 1, generator=g)
        if r % 3 == 0:                                   # 480 equal ones, an entry to a vector
            z[r, 8 * at[:480] + 5] = 4.0
        elif r % 3 == 1:                                 # 60 vectors full of different ones
            full = (8 * at[:60, None] + torch.arange(8)).reshape(-1)
            z[r, full] = 2.0 + torch.randperm(480, generator=g).float() / 64
        else:                                            # equal ones beyond all room
            z[r, ::2] = 3.0
    z = z.to(dtype)
    t = C.make_targets((rows, v), None, 2, g)
    z, t = z.to(dev), t.to(dev)
    for k in (1, 8, 40):
        for _ in range(3):
            out = cb.profile_log_probs(z, t, top_k=k)
        C.check_scores(z, out, t, k, None, None, 1.0)
