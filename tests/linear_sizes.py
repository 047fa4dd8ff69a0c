"""Sizes of fp8 products for every form that the plan has, on 256 CUs: (rows, inputs, outputs) of each, the smallest
found with six blocks or more to a workgroup (so that every LDS slot is filled again), rows and outputs that fill no tile."""

# (outputs, rows of a tile, inputs split): sizes whose last block of 128 inputs is whole, and others
TILES = {
    (16, 16, False): [(1, 768, 66), (13, 2048, 1001), (1, 784, 65), (11, 2032, 4093)],
    (16, 32, False): [(17, 896, 66), (31, 2560, 3001), (17, 784, 68), (29, 1008, 4001)],
    (16, 64, False): [(35, 768, 73), (61, 1024, 2003), (33, 800, 66), (63, 912, 1999)],
    (32, 16, False): [(1, 768, 4135), (5, 1024, 6001), (1, 784, 4147), (7, 1040, 8003)],
    (32, 32, False): [(17, 768, 4450), (18, 800, 4115)],
    (32, 64, False): [(36, 768, 4411), (34, 816, 4249)],
    (128, 64, False): [(69, 768, 4277), (65, 800, 4191), (333, 2000, 4999)],
    (128, 64, True): [(20, 10240, 70), (18, 9088, 65), (18, 8944, 66), (17, 9056, 67)],
    (128, 128, False): [(5713, 768, 268), (5461, 784, 265), (475, 4416, 5014)],
    (128, 128, True): [(69, 3200, 5631), (65, 4736, 4459), (65, 3536, 4213), (65, 4256, 4418)],
    (256, 128, False): [(529, 768, 6735), (6966, 784, 531)],
    (256, 128, True): [(4531, 5376, 135), (4182, 5120, 139), (2715, 7952, 129), (2717, 7760, 130)],
    (256, 256, False): [(3678, 768, 2181), (1666, 784, 4647), (6063, 2480, 5371)],
    (256, 256, True): [(5926, 9600, 315), (6190, 8832, 269), (6006, 8288, 274), (5477, 8752, 270)],
}
# rows of 16 bits that every workgroup quantises itself
OWN = {16: [(1, 768, 66), (3, 5120, 576), (1, 784, 65), (16, 1008, 2001)], 32: [(1, 768, 4135), (9, 1024, 8001), (5, 784, 4147)]}


def all_sizes():
    return sorted({s for sizes in [*TILES.values(), *OWN.values()] for s in sizes}, key=lambda s: s[0] * s[1] * s[2])
