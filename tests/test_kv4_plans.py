"""CPU test of the arithmetic that cuts attention over the 4-bit cache into
parts (steps_per_part in csrc/kv4.hip), replayed in 32 bits as the device does
it: whatever the lengths, the records fit the workspace that the library asks
for by shapes alone, and the units fit blocks + places."""

import random

import numpy as np
import pytest

F = np.float32
REC_BYTES = (2048 + 32) * 4  # of 16 rows


def _lib():
    from swarmlora_amd import _lib
    return _lib.load()


def steps_per_part(rb, steps, hkv, slots, min_spp):
    """rb, steps: blocks and steps of every sequence."""
    mine = [F(b) * F(hkv) for b in rb]
    lanes = [F(0)] * 64
    for i, (m, st) in enumerate(zip(mine, steps)):
        lanes[i % 64] += m * F(st)

    def total(v):
        s = F(0)
        for x in v:
            s += F(x)
        return s
    all_ = total(lanes) * F(1.0001)
    lo = max(min_spp, int(min(all_ / F(slots) + F(1), F(2.0 ** 30))))
    if len(rb) > 64:
        return lo

    def units(spp):
        return total(m * np.ceil(F(st) / F(spp)) for m, st in zip(mine, steps))
    blocks = total(mine)
    if blocks >= slots or units(lo) <= slots:
        return lo
    hi = max(lo, int(min(all_ / (F(slots) - blocks) + F(1), F(2.0 ** 30))))
    while hi - lo > max(1, lo >> 4):
        mid = (lo + hi) >> 1
        if units(mid) <= slots:
            hi = mid
        else:
            lo = mid
    return hi


# rows of a block, keys of a step, places, least steps of a part, new tokens (of
# four heads: up to 16, 64 and more rows)
KINDS = {"one": (16, 32, 1024, 16, (1, 1)), "drafts": (32, 32, 512, 16, (5, 16)), "prompts": (128, 64, 512, 8, (33, 3000))}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("many", [False, True])
def test_units_and_records_stay_within_their_bounds(kind, many):
    rows, keys, slots, min_spp, span = KINDS[kind]
    rng = random.Random(f"{kind}{many}")
    seen = set()
    for _ in range(150):
        nseq = rng.randrange(65, 300) if many else int(2 ** rng.uniform(0, 6))
        hkv, G = rng.choice([1, 2, 4, 8, 32]), 4
        top = int(2 ** rng.uniform(6, 20))
        ctx = [int(2 ** rng.uniform(0, np.log2(top))) if rng.random() < 0.7 else top for _ in range(nseq)]
        L = rng.randint(*span)  # the uniform form: one kernel for all of them
        max_keys = (max(ctx) + L + 15) // 16 * 16 + (0 if kind != "prompts" else 1 << 21)
        ws = _lib().swl_kv4_attention_workspace(nseq, nseq * L, 0, L, G * hkv, hkv, max_keys)
        rb = [(L * G + rows - 1) // rows] * nseq
        steps = [max(1, (c + L + keys - 1) // keys) for c in ctx]
        spp = steps_per_part(rb, steps, hkv, slots, min_spp)
        parts = [(s + spp - 1) // spp for s in steps]
        blocks = sum(rb) * hkv
        units = sum(b * p for b, p in zip(rb, parts)) * hkv
        cut = sum(b for b, p in zip(rb, parts) if p > 1) * hkv
        recs = sum(b * p for b, p in zip(rb, parts) if p > 1) * hkv
        assert units <= blocks + slots and cut <= slots and recs <= 2 * slots
        assert recs * (rows // 16) * REC_BYTES <= ws
        if nseq <= 64 and blocks < slots and spp > min_spp:
            assert units <= slots
        seen.add((spp > min_spp, blocks >= slots, units > slots, recs > 0))
    assert len(seen) >= 3  # the branches are met
