"""The index arrays of a prefill step, entry by entry from their definition."""
PAGE = 32


def naive(new, history, slots, table, window=0, sinks=0):
    out = {n: [] for n in ("seq_lens", "job_seq", "job_page", "page_blk", "page_dst", "tail_blk", "tail_info", "new_dst", "slot_map")}
    out["q_start"], out["key_start"] = [0], [0]
    for r, (t, h) in enumerate(zip(new, history)):
        key = out["key_start"][-1]
        first = -(-sinks // PAGE)
        begin = max(0, h - window + 1) // PAGE if window else 0             # the page of the first new token's window
        for p in range(-(-h // PAGE)):
            if window and first <= p < begin:
                continue
            if (p + 1) * PAGE <= h:
                out["page_blk"].append(table[r][p])
                out["page_dst"].append(key)
                key += PAGE
            else:
                out["tail_blk"].append(table[r][p])
                out["tail_info"].append([key, h - p * PAGE, slots[r]])
                key += h - p * PAGE
        for p in sorted({(h + i) // PAGE for i in range(t)}):
            out["job_seq"].append(r)
            out["job_page"].append(p)
        for i in range(t):
            out["new_dst"].append(key + i)
            out["slot_map"].append(table[r][(h + i) // PAGE] * PAGE + (h + i) % PAGE)
        out["q_start"].append(out["q_start"][-1] + t)
        out["key_start"].append(key + t)
        out["seq_lens"].append(h + t)
    return out


def check(kk, torch, new, history, device, window=0, sinks=0, spare=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    R = len(new)
    cols = max([-(-(t + h) // PAGE) for t, h in zip(new, history)], default=0) + spare
    table = torch.randint(0, 1 << 26, (R, cols), generator=g, dtype=torch.int32)
    slots = torch.randperm(R + 3, generator=g)[:R].to(torch.int32)
    sizes = kk.map_sizes(new, history, window=window or None, sinks=sinks)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).to(device)  # noqa: E731
    got = kk.step_maps(i32(new), i32(history), slots.to(device), table.to(device), sizes)
    want = naive(new, history, slots.tolist(), table.tolist(), window, sinks)
    for name, x in want.items():
        y = getattr(got, name)
        assert y.tolist() == x, name
        assert y.dtype == (torch.int64 if name == "slot_map" else torch.int32) and y.is_contiguous()
    assert sizes.keys == want["key_start"][-1]
    return got
