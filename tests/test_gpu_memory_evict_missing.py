"""What an eviction leaves of a stream some of whose pages are not there, by the tokens' positions."""
import pytest
import torch

import d2conv3d_amd as d2c

pytestmark = pytest.mark.gpu

SLOTS, PAGE, KEEP, RECENT = 20, 4, 8, 2
READ_MOST = (1, 3, 9, 12, 13, 17)      # (and the newest, 18 and 19, which were read least)


def stream(missing, dtype, dev):
    """One stream of 20 tokens in 5 pages, token i in slot i, `missing` of the pages' numbers outside the pool; a token's key and value are its position."""
    table = torch.tensor([[4, 2, 0, 3, 1]], dtype=torch.int32)
    m = d2c.PagedMemory.empty(1, SLOTS, 2, 8, page=PAGE, dtype=dtype, device=dev)
    slot = torch.arange(SLOTS)
    page, place = table[0].long()[slot // PAGE].to(dev), (slot % PAGE).to(dev)
    m.positions[page, :, place] = slot.int()[:, None].to(dev)
    m.key[page, :, place] = slot[:, None, None].to(dev, dtype)
    m.value[page, :, place] = -slot[:, None, None].to(dev, dtype)
    usage = torch.tensor([1.0 + i / 100 if i in READ_MOST else 0.0 if i >= 18 else 0.5 - i / 100 for i in range(SLOTS)])
    m.usage[page, :, place] = usage[:, None].to(dev)
    m.lengths.fill_(SLOTS)
    m.seen.fill_(SLOTS)
    for i, number in missing:
        table[0, i] = number
    m.table.copy_(table)
    return m


def tokens(m):
    """Positions in the slots that are there after it, None in those that are not, the same in both heads."""
    found = []
    for s in range(int(m.lengths[0])):
        page = int(m.table[0, s // PAGE])
        if not 0 <= page < m.key.shape[0]:
            found.append(None)
            continue
        at = m.positions[page, :, s % PAGE].tolist()
        assert at[0] == at[1]
        assert bool((m.key[page, :, s % PAGE] == at[0]).all()) and bool((m.value[page, :, s % PAGE] == -at[0]).all())
        found.append(at[0])
    return found


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_before_keep(dtype, dev):
    """Slots 4 to 7 are not there: they go, with slots 0 and 2, and the six tokens from behind come in order -- 9 and 12 into 0 and 2, the others, the newest among them, nowhere."""
    m = stream([(1, -1)], dtype, dev)
    m.evict(KEEP, RECENT)
    assert tokens(m) == [9, 1, 12, 3, None, None, None, None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_behind_keep(dtype, dev):
    """Slots 12 to 15 are not there: nothing that is there is lost but what was read least."""
    m = stream([(3, 99)], dtype, dev)
    m.evict(KEEP, RECENT)
    # (12 and 13 are gone with their page: 0 and 2, of the largest usage beside those, stay where they are; 9, 17, 18, 19 go into 4 .. 7)
    assert tokens(m) == [0, 1, 2, 3, 9, 17, 18, 19]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_pages(dtype, dev):
    m = stream([], dtype, dev)
    m.evict(KEEP, RECENT)
    assert tokens(m) == [9, 1, 12, 3, 13, 17, 18, 19]
