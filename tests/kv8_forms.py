"""Attention calls by the kernel that the plan takes for them (256 CUs)."""

# nq, H, D, page, rows, past, window, max_pages, kernel: tables with room for codes that the last-level cache does not hold
STREAMS = [
    (8, 8, 64, 64, [1, 1], [700, 33], 0, 3000, "gh_kv8_attn_l1s_k"),
    (4, 4, 48, 32, [2, 1], [200, 900], 0, 20000, "gh_kv8_attn_l1rs_k"),
    (3, 1, 16, 16, [1], [300], 0, 260000, "gh_kv8_attn_l1rs_k"),
    (8, 4, 128, 32, [1, 3], [500, 61], 0, 7000, "gh_kv8_attn_l2s_k"),
    (12, 4, 96, 64, [2], [333], 0, 8000, "gh_kv8_attn_l2rs_k"),
    (16, 8, 256, 32, [1, 5, 0], [400, 31, 7], 0, 2000, "gh_kv8_attn_l4s_k"),
    (6, 2, 144, 16, [1], [640], 0, 24000, "gh_kv8_attn_l4rs_k"),
    (4, 2, 192, 32, [3, 1], [97, 500], 0, 8000, "gh_kv8_attn_l4rs_k"),
    (8, 2, 512, 64, [1, 2], [450, 40], 0, 2000, "gh_kv8_attn_l8s_k"),
    (5, 1, 400, 32, [1], [600], 0, 9000, "gh_kv8_attn_l8rs_k"),
    (3, 1, 272, 16, [2], [35], 0, 30000, "gh_kv8_attn_l8rs_k"),
    # a window that is itself so long
    (8, 8, 64, 64, [1, 1], [700, 33], 1000000, 3000, "gh_kv8_attn_l1s_k"),
    (12, 4, 96, 64, [2], [333], 2000000000, 8000, "gh_kv8_attn_l2rs_k"),
]

# nq, H, D, page, rows, past, window, (num_rows, max_rows), kernel: tiles for every CU
PROMPTS = [
    (8, 8, 64, 32, [1100], [0], 0, (1100, 1100), "gh_kv8_rows_l1_k"),
    (8, 8, 48, 32, [1100], [0], 0, (1100, 1100), "gh_kv8_rows_l1r_k"),
    (8, 8, 128, 64, [1050], [3], 40, (1050, 1050), "gh_kv8_rows_l2_k"),
    (8, 8, 112, 64, [1030], [50], 0, (1030, 1030), "gh_kv8_rows_l2r_k"),
    (16, 8, 256, 64, [520], [0], 0, (520, 520), "gh_kv8_rows_l4_k"),
    (16, 8, 144, 32, [530], [9], 0, (530, 530), "gh_kv8_rows_l4r_k"),
    (8, 4, 192, 16, [1040], [0], 77, (1040, 1040), "gh_kv8_rows_l4r_k"),
    (8, 2, 512, 64, [1030], [0], 0, (1030, 1030), "gh_kv8_rows_l8_k"),
    (16, 4, 400, 32, [540], [1], 0, (540, 540), "gh_kv8_rows_l8r_k"),
    # bounds below and above the rows that there are
    (8, 8, 64, 32, [900, 30, 500], [0, 5, 70], 0, (1200, 700), "gh_kv8_rows_l1_k"),
    (8, 8, 64, 32, [900, 30, 500], [0, 5, 70], 50, (905, 2000), "gh_kv8_rows_l1_k"),
    (16, 8, 256, 32, [600, 40], [0, 5], 0, (620, 590), "gh_kv8_rows_l4_k"),
    (16, 8, 256, 32, [300, 40], [0, 5], 0, (340, 300), "gh_kv8_rows_l4_k"),
]
