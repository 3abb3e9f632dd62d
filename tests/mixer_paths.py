"""Shapes whose calls take the paths of long and of many sequences: a thread of the convolution that slides its window over several runs, scan workgroups that walk
many tiles (wide tiles, and narrow ones of more workgroups than CUs), a workgroup of the norm's backward that takes several rows.  test_mixer_paths_cpu.py
checks that they do, test_mixer_paths_gpu.py their results."""

# (B, L, D, K)
CONV = [(600, 70, 260, K) for K in range(1, 9)] + [(8, 1031, 1030, 4), (8, 1031, 1030, 8), (16, 40001, 3, 5)]

# (B, L, D, N, G): 129 to 256 workgroups of up to 16 states
SCAN_WIDE = [(9, 1000, 250, 16, 1), (10, 700, 237, 8, 3), (8, 515, 260, 5, 1), (16, 960, 256, 16, 1)]
# ... more than 256
SCAN_MANY = [(9, 500, 480, 16, 3), (9, 401, 470, 8, 1), (9, 300, 480, 32, 1), (9, 150, 466, 64, 1), (16, 70, 300, 16, 1), (18, 270, 240, 11, 1)]

# (rows, C, type)
NORM = [(2600, 1999, 'f32'), (2600, 1999, 'bf16'), (2600, 2000, 'f16'), (1500, 4095, 'f32'), (700, 8191, 'f32'), (700, 8191, 'bf16'), (700, 12001, 'f16'), (20011, 48, 'f32'),
        (17003, 127, 'bf16'), (5003, 320, 'f32'), (5003, 1021, 'bf16'), (600, 9001, 'f32'), (600, 16400, 'bf16')]
