// Generated by gen_tile_asm.py mx -- do not edit; see that file for the register plan and the schedule.
#pragma once
#define SK_TILE_ASM_LOOP_MX \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "v_accvgpr_write_b32 a128, 0\n\t" \
  "v_accvgpr_write_b32 a129, 0\n\t" \
  "v_accvgpr_write_b32 a130, 0\n\t" \
  "v_accvgpr_write_b32 a131, 0\n\t" \
  "v_accvgpr_write_b32 a132, 0\n\t" \
  "v_accvgpr_write_b32 a133, 0\n\t" \
  "v_accvgpr_write_b32 a134, 0\n\t" \
  "v_accvgpr_write_b32 a135, 0\n\t" \
  "v_accvgpr_write_b32 a136, 0\n\t" \
  "v_accvgpr_write_b32 a137, 0\n\t" \
  "v_accvgpr_write_b32 a138, 0\n\t" \
  "v_accvgpr_write_b32 a139, 0\n\t" \
  "v_accvgpr_write_b32 a140, 0\n\t" \
  "v_accvgpr_write_b32 a141, 0\n\t" \
  "v_accvgpr_write_b32 a142, 0\n\t" \
  "v_accvgpr_write_b32 a143, 0\n\t" \
  "v_accvgpr_write_b32 a144, 0\n\t" \
  "v_accvgpr_write_b32 a145, 0\n\t" \
  "v_accvgpr_write_b32 a146, 0\n\t" \
  "v_accvgpr_write_b32 a147, 0\n\t" \
  "v_accvgpr_write_b32 a148, 0\n\t" \
  "v_accvgpr_write_b32 a149, 0\n\t" \
  "v_accvgpr_write_b32 a150, 0\n\t" \
  "v_accvgpr_write_b32 a151, 0\n\t" \
  "v_accvgpr_write_b32 a152, 0\n\t" \
  "v_accvgpr_write_b32 a153, 0\n\t" \
  "v_accvgpr_write_b32 a154, 0\n\t" \
  "v_accvgpr_write_b32 a155, 0\n\t" \
  "v_accvgpr_write_b32 a156, 0\n\t" \
  "v_accvgpr_write_b32 a157, 0\n\t" \
  "v_accvgpr_write_b32 a158, 0\n\t" \
  "v_accvgpr_write_b32 a159, 0\n\t" \
  "v_accvgpr_write_b32 a160, 0\n\t" \
  "v_accvgpr_write_b32 a161, 0\n\t" \
  "v_accvgpr_write_b32 a162, 0\n\t" \
  "v_accvgpr_write_b32 a163, 0\n\t" \
  "v_accvgpr_write_b32 a164, 0\n\t" \
  "v_accvgpr_write_b32 a165, 0\n\t" \
  "v_accvgpr_write_b32 a166, 0\n\t" \
  "v_accvgpr_write_b32 a167, 0\n\t" \
  "v_accvgpr_write_b32 a168, 0\n\t" \
  "v_accvgpr_write_b32 a169, 0\n\t" \
  "v_accvgpr_write_b32 a170, 0\n\t" \
  "v_accvgpr_write_b32 a171, 0\n\t" \
  "v_accvgpr_write_b32 a172, 0\n\t" \
  "v_accvgpr_write_b32 a173, 0\n\t" \
  "v_accvgpr_write_b32 a174, 0\n\t" \
  "v_accvgpr_write_b32 a175, 0\n\t" \
  "v_accvgpr_write_b32 a176, 0\n\t" \
  "v_accvgpr_write_b32 a177, 0\n\t" \
  "v_accvgpr_write_b32 a178, 0\n\t" \
  "v_accvgpr_write_b32 a179, 0\n\t" \
  "v_accvgpr_write_b32 a180, 0\n\t" \
  "v_accvgpr_write_b32 a181, 0\n\t" \
  "v_accvgpr_write_b32 a182, 0\n\t" \
  "v_accvgpr_write_b32 a183, 0\n\t" \
  "v_accvgpr_write_b32 a184, 0\n\t" \
  "v_accvgpr_write_b32 a185, 0\n\t" \
  "v_accvgpr_write_b32 a186, 0\n\t" \
  "v_accvgpr_write_b32 a187, 0\n\t" \
  "v_accvgpr_write_b32 a188, 0\n\t" \
  "v_accvgpr_write_b32 a189, 0\n\t" \
  "v_accvgpr_write_b32 a190, 0\n\t" \
  "v_accvgpr_write_b32 a191, 0\n\t" \
  "v_accvgpr_write_b32 a192, 0\n\t" \
  "v_accvgpr_write_b32 a193, 0\n\t" \
  "v_accvgpr_write_b32 a194, 0\n\t" \
  "v_accvgpr_write_b32 a195, 0\n\t" \
  "v_accvgpr_write_b32 a196, 0\n\t" \
  "v_accvgpr_write_b32 a197, 0\n\t" \
  "v_accvgpr_write_b32 a198, 0\n\t" \
  "v_accvgpr_write_b32 a199, 0\n\t" \
  "v_accvgpr_write_b32 a200, 0\n\t" \
  "v_accvgpr_write_b32 a201, 0\n\t" \
  "v_accvgpr_write_b32 a202, 0\n\t" \
  "v_accvgpr_write_b32 a203, 0\n\t" \
  "v_accvgpr_write_b32 a204, 0\n\t" \
  "v_accvgpr_write_b32 a205, 0\n\t" \
  "v_accvgpr_write_b32 a206, 0\n\t" \
  "v_accvgpr_write_b32 a207, 0\n\t" \
  "v_accvgpr_write_b32 a208, 0\n\t" \
  "v_accvgpr_write_b32 a209, 0\n\t" \
  "v_accvgpr_write_b32 a210, 0\n\t" \
  "v_accvgpr_write_b32 a211, 0\n\t" \
  "v_accvgpr_write_b32 a212, 0\n\t" \
  "v_accvgpr_write_b32 a213, 0\n\t" \
  "v_accvgpr_write_b32 a214, 0\n\t" \
  "v_accvgpr_write_b32 a215, 0\n\t" \
  "v_accvgpr_write_b32 a216, 0\n\t" \
  "v_accvgpr_write_b32 a217, 0\n\t" \
  "v_accvgpr_write_b32 a218, 0\n\t" \
  "v_accvgpr_write_b32 a219, 0\n\t" \
  "v_accvgpr_write_b32 a220, 0\n\t" \
  "v_accvgpr_write_b32 a221, 0\n\t" \
  "v_accvgpr_write_b32 a222, 0\n\t" \
  "v_accvgpr_write_b32 a223, 0\n\t" \
  "v_accvgpr_write_b32 a224, 0\n\t" \
  "v_accvgpr_write_b32 a225, 0\n\t" \
  "v_accvgpr_write_b32 a226, 0\n\t" \
  "v_accvgpr_write_b32 a227, 0\n\t" \
  "v_accvgpr_write_b32 a228, 0\n\t" \
  "v_accvgpr_write_b32 a229, 0\n\t" \
  "v_accvgpr_write_b32 a230, 0\n\t" \
  "v_accvgpr_write_b32 a231, 0\n\t" \
  "v_accvgpr_write_b32 a232, 0\n\t" \
  "v_accvgpr_write_b32 a233, 0\n\t" \
  "v_accvgpr_write_b32 a234, 0\n\t" \
  "v_accvgpr_write_b32 a235, 0\n\t" \
  "v_accvgpr_write_b32 a236, 0\n\t" \
  "v_accvgpr_write_b32 a237, 0\n\t" \
  "v_accvgpr_write_b32 a238, 0\n\t" \
  "v_accvgpr_write_b32 a239, 0\n\t" \
  "v_accvgpr_write_b32 a240, 0\n\t" \
  "v_accvgpr_write_b32 a241, 0\n\t" \
  "v_accvgpr_write_b32 a242, 0\n\t" \
  "v_accvgpr_write_b32 a243, 0\n\t" \
  "v_accvgpr_write_b32 a244, 0\n\t" \
  "v_accvgpr_write_b32 a245, 0\n\t" \
  "v_accvgpr_write_b32 a246, 0\n\t" \
  "v_accvgpr_write_b32 a247, 0\n\t" \
  "v_accvgpr_write_b32 a248, 0\n\t" \
  "v_accvgpr_write_b32 a249, 0\n\t" \
  "v_accvgpr_write_b32 a250, 0\n\t" \
  "v_accvgpr_write_b32 a251, 0\n\t" \
  "v_accvgpr_write_b32 a252, 0\n\t" \
  "v_accvgpr_write_b32 a253, 0\n\t" \
  "v_accvgpr_write_b32 a254, 0\n\t" \
  "v_accvgpr_write_b32 a255, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_add_u32 s81, %[ga0], 128\n\t" \
  "s_add_u32 s82, %[gb0], 128\n\t" \
  "s_mov_b32 s88, %[el]\n\t" \
  "s_mov_b32 s89, %[eka]\n\t" \
  "s_mov_b32 s90, %[ekb]\n\t" \
  "v_xor_b32 v124, 16, %[ra0]\n\t" \
  "v_xor_b32 v125, 16, %[rb0]\n\t" \
  "v_mov_b32 v126, %[rda]\n\t" \
  "v_mov_b32 v127, %[rdb]\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "s_add_u32 s87, s87, 1\n\t" \
  "s_cmp_eq_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s85, 0x80000000, 0\n\t" \
  "v_and_b32 v122, s85, %[tail]\n\t" \
  "v_or3_b32 v120, s84, %[voa], v122\n\t" \
  "v_or3_b32 v121, s84, %[vob], v122\n\t" \
  "s_waitcnt vmcnt(8)\n\t" \
  "s_barrier\n\t" \
  "ds_read_u16 v88, v126 offset:0\n\t" \
  "ds_read_u16 v89, v126 offset:256\n\t" \
  "ds_read_u16 v90, v126 offset:512\n\t" \
  "ds_read_u16 v91, v126 offset:768\n\t" \
  "ds_read_u16 v92, v126 offset:1024\n\t" \
  "ds_read_u16 v93, v126 offset:1280\n\t" \
  "ds_read_u16 v94, v126 offset:1536\n\t" \
  "ds_read_u16 v95, v126 offset:1792\n\t" \
  "ds_read_u16 v96, v127 offset:0\n\t" \
  "ds_read_u16 v97, v127 offset:256\n\t" \
  "ds_read_u16 v98, v127 offset:512\n\t" \
  "ds_read_u16 v99, v127 offset:768\n\t" \
  "ds_read_u16 v100, v127 offset:1024\n\t" \
  "ds_read_u16 v101, v127 offset:1280\n\t" \
  "ds_read_u16 v102, v127 offset:1536\n\t" \
  "ds_read_u16 v103, v127 offset:1792\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[160:163], v[128:131], a[0:3], v96, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[176:179], %[rb0] offset:8192\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[164:167], v[128:131], a[4:7], v97, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[180:183], %[rb0] offset:10240\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[168:171], v[128:131], a[8:11], v98, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[184:187], %[rb0] offset:12288\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[172:175], v[128:131], a[12:15], v99, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[188:191], %[rb0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[172:175], v[132:135], a[44:47], v99, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[144:147], %[ra0] offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[168:171], v[132:135], a[40:43], v98, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[148:151], %[ra0] offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[164:167], v[132:135], a[36:39], v97, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[152:155], %[ra0] offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[160:163], v[132:135], a[32:35], v96, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[156:159], %[ra0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[160:163], v[136:139], a[64:67], v96, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s81, %[gas2]\n\t" \
  "s_add_u32 m0, s86, 8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[164:167], v[136:139], a[68:71], v97, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[192:195], v124 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[168:171], v[136:139], a[72:75], v98, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[172:175], v[136:139], a[76:79], v99, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v104, v126 offset:8\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[172:175], v[140:143], a[108:111], v99, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[168:171], v[140:143], a[104:107], v98, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[164:167], v[140:143], a[100:103], v97, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[224:227], v125 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[160:163], v[140:143], a[96:99], v96, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v105, v126 offset:264\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[176:179], v[140:143], a[112:115], v100, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[180:183], v[140:143], a[116:119], v101, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[184:187], v[140:143], a[120:123], v102, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 24576\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[188:191], v[140:143], a[124:127], v103, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[188:191], v[136:139], a[92:95], v103, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[228:231], v125 offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[184:187], v[136:139], a[88:91], v102, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[180:183], v[136:139], a[84:87], v101, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v106, v126 offset:520\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[176:179], v[136:139], a[80:83], v100, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[176:179], v[132:135], a[48:51], v100, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 28672\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[180:183], v[132:135], a[52:55], v101, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[232:235], v125 offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[184:187], v[132:135], a[56:59], v102, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[188:191], v[132:135], a[60:63], v103, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v107, v126 offset:776\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[188:191], v[128:131], a[28:31], v103, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[184:187], v[128:131], a[24:27], v102, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s82, %[gbs2]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[180:183], v[128:131], a[20:23], v101, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[176:179], v[128:131], a[16:19], v100, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[236:239], v125 offset:6144\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[144:147], v[176:179], v[144:147], a[144:147], v100, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[148:151], v[180:183], v[144:147], a[148:151], v101, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v108, v126 offset:1032\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[152:155], v[184:187], v[144:147], a[152:155], v102, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[156:159], v[188:191], v[144:147], a[156:159], v103, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[188:191], v[188:191], v[148:151], a[188:191], v103, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[196:199], v124 offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[184:187], v[184:187], v[148:151], a[184:187], v102, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[180:183], v[180:183], v[148:151], a[180:183], v101, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v109, v126 offset:1288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[176:179], v[176:179], v[148:151], a[176:179], v100, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[208:211], v[176:179], v[152:155], a[208:211], v100, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[212:215], v[180:183], v[152:155], a[212:215], v101, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[216:219], v[184:187], v[152:155], a[216:219], v102, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[200:203], v124 offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[220:223], v[188:191], v[152:155], a[220:223], v103, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[252:255], v[188:191], v[156:159], a[252:255], v103, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v110, v126 offset:1544\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[248:251], v[184:187], v[156:159], a[248:251], v102, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[244:247], v[180:183], v[156:159], a[244:247], v101, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[240:243], v[176:179], v[156:159], a[240:243], v100, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[204:207], v124 offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[236:239], v[172:175], v[156:159], a[236:239], v99, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[232:235], v[168:171], v[156:159], a[232:235], v98, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v111, v126 offset:1800\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[228:231], v[164:167], v[156:159], a[228:231], v97, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[224:227], v[160:163], v[156:159], a[224:227], v96, v95 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 m0, s88\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[192:195], v[160:163], v[152:155], a[192:195], v96, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[196:199], v[164:167], v[152:155], a[196:199], v97, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 %[ve], %[rea], s89 offen lds\n\t" \
  "s_add_u32 s89, s89, %[esa]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[200:203], v[168:171], v[152:155], a[200:203], v98, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[204:207], v[172:175], v[152:155], a[204:207], v99, v94 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[172:175], v[172:175], v[148:151], a[172:175], v99, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 m0, s88, 4096\n\t" \
  "s_xor_b32 s88, s88, 0x2000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[168:171], v[168:171], v[148:151], a[168:171], v98, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[164:167], v[164:167], v[148:151], a[164:167], v97, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[160:163], v[160:163], v[148:151], a[160:163], v96, v93 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 %[ve], %[reb], s90 offen lds\n\t" \
  "s_add_u32 s90, s90, %[esb]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[128:131], v[160:163], v[144:147], a[128:131], v96, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[132:135], v[164:167], v[144:147], a[132:135], v97, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[136:139], v[168:171], v[144:147], a[136:139], v98, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[140:143], v[172:175], v[144:147], a[140:143], v99, v92 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt vmcnt(10) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[224:227], v[192:195], a[0:3], v96, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[240:243], v125 offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[228:231], v[192:195], a[4:7], v97, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[244:247], v125 offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[232:235], v[192:195], a[8:11], v98, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[248:251], v125 offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[236:239], v[192:195], a[12:15], v99, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[252:255], v125 offset:14336\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[236:239], v[196:199], a[44:47], v99, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[208:211], v124 offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[232:235], v[196:199], a[40:43], v98, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[212:215], v124 offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[228:231], v[196:199], a[36:39], v97, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[216:219], v124 offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[224:227], v[196:199], a[32:35], v96, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[220:223], v124 offset:14336\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[224:227], v[200:203], a[64:67], v96, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, 128\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[228:231], v[200:203], a[68:71], v97, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[232:235], v[200:203], a[72:75], v98, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s87, s87, 1\n\t" \
  "s_cmp_eq_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s85, 0x80000000, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[236:239], v[200:203], a[76:79], v99, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_and_b32 v122, s85, %[tail]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[236:239], v[204:207], a[108:111], v99, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_or3_b32 v120, s84, %[voa], v122\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[232:235], v[204:207], a[104:107], v98, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_or3_b32 v121, s84, %[vob], v122\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[228:231], v[204:207], a[100:103], v97, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[224:227], v[204:207], a[96:99], v96, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[240:243], v[204:207], a[112:115], v100, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v112, v127 offset:8\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[244:247], v[204:207], a[116:119], v101, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[248:251], v[204:207], a[120:123], v102, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v124, 0x10000, v124\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[252:255], v[204:207], a[124:127], v103, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[252:255], v[200:203], a[92:95], v103, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[248:251], v[200:203], a[88:91], v102, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v113, v127 offset:264\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[244:247], v[200:203], a[84:87], v101, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[240:243], v[200:203], a[80:83], v100, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[240:243], v[196:199], a[48:51], v100, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[244:247], v[196:199], a[52:55], v101, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v114, v127 offset:520\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[248:251], v[196:199], a[56:59], v102, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[252:255], v[196:199], a[60:63], v103, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[252:255], v[192:195], a[28:31], v103, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[248:251], v[192:195], a[24:27], v102, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[244:247], v[192:195], a[20:23], v101, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v115, v127 offset:776\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[240:243], v[192:195], a[16:19], v100, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[144:147], v[240:243], v[208:211], a[144:147], v100, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[148:151], v[244:247], v[208:211], a[148:151], v101, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[152:155], v[248:251], v[208:211], a[152:155], v102, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[156:159], v[252:255], v[208:211], a[156:159], v103, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[188:191], v[252:255], v[212:215], a[188:191], v103, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v116, v127 offset:1032\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[184:187], v[248:251], v[212:215], a[184:187], v102, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[180:183], v[244:247], v[212:215], a[180:183], v101, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[176:179], v[240:243], v[212:215], a[176:179], v100, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[208:211], v[240:243], v[216:219], a[208:211], v100, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v117, v127 offset:1288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[212:215], v[244:247], v[216:219], a[212:215], v101, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[216:219], v[248:251], v[216:219], a[216:219], v102, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[220:223], v[252:255], v[216:219], a[220:223], v103, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[252:255], v[252:255], v[220:223], a[252:255], v103, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[248:251], v[248:251], v[220:223], a[248:251], v102, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v118, v127 offset:1544\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[244:247], v[244:247], v[220:223], a[244:247], v101, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[240:243], v[240:243], v[220:223], a[240:243], v100, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[236:239], v[236:239], v[220:223], a[236:239], v99, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[232:235], v[232:235], v[220:223], a[232:235], v98, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v119, v127 offset:1800\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[228:231], v[228:231], v[220:223], a[228:231], v97, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[224:227], v[224:227], v[220:223], a[224:227], v96, v95 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v125, 0x10000, v125\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[192:195], v[224:227], v[216:219], a[192:195], v96, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[196:199], v[228:231], v[216:219], a[196:199], v97, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[200:203], v[232:235], v[216:219], a[200:203], v98, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[204:207], v[236:239], v[216:219], a[204:207], v99, v94 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[172:175], v[236:239], v[212:215], a[172:175], v99, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[168:171], v[232:235], v[212:215], a[168:171], v98, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[164:167], v[228:231], v[212:215], a[164:167], v97, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[160:163], v[224:227], v[212:215], a[160:163], v96, v93 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[128:131], v[224:227], v[208:211], a[128:131], v96, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[132:135], v[228:231], v[208:211], a[132:135], v97, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[136:139], v[232:235], v[208:211], a[136:139], v98, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[140:143], v[236:239], v[208:211], a[140:143], v99, v92 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc0 L_sk_end%=\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[160:163], v[128:131], a[0:3], v112, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[176:179], %[rb0] offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[164:167], v[128:131], a[4:7], v113, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[180:183], %[rb0] offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[168:171], v[128:131], a[8:11], v114, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[184:187], %[rb0] offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[172:175], v[128:131], a[12:15], v115, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[188:191], %[rb0] offset:14336\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[172:175], v[132:135], a[44:47], v115, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[144:147], %[ra0] offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[168:171], v[132:135], a[40:43], v114, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[148:151], %[ra0] offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[164:167], v[132:135], a[36:39], v113, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[152:155], %[ra0] offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[160:163], v[132:135], a[32:35], v112, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[156:159], %[ra0] offset:14336\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[160:163], v[136:139], a[64:67], v112, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v126, 0x2000, v126\n\t" \
  "v_xor_b32 v127, 0x2000, v127\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[164:167], v[136:139], a[68:71], v113, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s81, %[gas2]\n\t" \
  "s_add_u32 m0, s86, 8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[168:171], v[136:139], a[72:75], v114, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[192:195], v124 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[172:175], v[136:139], a[76:79], v115, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v88, v126 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[172:175], v[140:143], a[108:111], v115, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[168:171], v[140:143], a[104:107], v114, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[164:167], v[140:143], a[100:103], v113, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[224:227], v125 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[160:163], v[140:143], a[96:99], v112, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 12288\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[176:179], v[140:143], a[112:115], v116, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v89, v126 offset:256\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[180:183], v[140:143], a[116:119], v117, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[184:187], v[140:143], a[120:123], v118, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[188:191], v[140:143], a[124:127], v119, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[188:191], v[136:139], a[92:95], v119, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[228:231], v125 offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[184:187], v[136:139], a[88:91], v118, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v90, v126 offset:512\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[180:183], v[136:139], a[84:87], v117, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 24576\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[176:179], v[136:139], a[80:83], v116, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[176:179], v[132:135], a[48:51], v116, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[180:183], v[132:135], a[52:55], v117, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[184:187], v[132:135], a[56:59], v118, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[232:235], v125 offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[188:191], v[132:135], a[60:63], v119, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v91, v126 offset:768\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[188:191], v[128:131], a[28:31], v119, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 28672\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[184:187], v[128:131], a[24:27], v118, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[180:183], v[128:131], a[20:23], v117, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[176:179], v[128:131], a[16:19], v116, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[236:239], v125 offset:6144\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[144:147], v[176:179], v[144:147], a[144:147], v116, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[148:151], v[180:183], v[144:147], a[148:151], v117, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v92, v126 offset:1024\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[152:155], v[184:187], v[144:147], a[152:155], v118, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[156:159], v[188:191], v[144:147], a[156:159], v119, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s82, %[gbs2]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[188:191], v[188:191], v[148:151], a[188:191], v119, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[184:187], v[184:187], v[148:151], a[184:187], v118, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[196:199], v124 offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[180:183], v[180:183], v[148:151], a[180:183], v117, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[176:179], v[176:179], v[148:151], a[176:179], v116, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v93, v126 offset:1280\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[208:211], v[176:179], v[152:155], a[208:211], v116, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[212:215], v[180:183], v[152:155], a[212:215], v117, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[216:219], v[184:187], v[152:155], a[216:219], v118, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[220:223], v[188:191], v[152:155], a[220:223], v119, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[200:203], v124 offset:4096\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[252:255], v[188:191], v[156:159], a[252:255], v119, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v94, v126 offset:1536\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[248:251], v[184:187], v[156:159], a[248:251], v118, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[244:247], v[180:183], v[156:159], a[244:247], v117, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[240:243], v[176:179], v[156:159], a[240:243], v116, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[236:239], v[172:175], v[156:159], a[236:239], v115, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[232:235], v[168:171], v[156:159], a[232:235], v114, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[204:207], v124 offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[228:231], v[164:167], v[156:159], a[228:231], v113, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v95, v126 offset:1792\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[224:227], v[160:163], v[156:159], a[224:227], v112, v111 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[192:195], v[160:163], v[152:155], a[192:195], v112, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[196:199], v[164:167], v[152:155], a[196:199], v113, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[200:203], v[168:171], v[152:155], a[200:203], v114, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[204:207], v[172:175], v[152:155], a[204:207], v115, v110 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[172:175], v[172:175], v[148:151], a[172:175], v115, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[168:171], v[168:171], v[148:151], a[168:171], v114, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[164:167], v[164:167], v[148:151], a[164:167], v113, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[160:163], v[160:163], v[148:151], a[160:163], v112, v109 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[128:131], v[160:163], v[144:147], a[128:131], v112, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[132:135], v[164:167], v[144:147], a[132:135], v113, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[136:139], v[168:171], v[144:147], a[136:139], v114, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[140:143], v[172:175], v[144:147], a[140:143], v115, v108 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[224:227], v[192:195], a[0:3], v112, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[240:243], v125 offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[228:231], v[192:195], a[4:7], v113, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[244:247], v125 offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[232:235], v[192:195], a[8:11], v114, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[248:251], v125 offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[236:239], v[192:195], a[12:15], v115, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[252:255], v125 offset:14336\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[236:239], v[196:199], a[44:47], v115, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[208:211], v124 offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[232:235], v[196:199], a[40:43], v114, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[212:215], v124 offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[228:231], v[196:199], a[36:39], v113, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[216:219], v124 offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[224:227], v[196:199], a[32:35], v112, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[220:223], v124 offset:14336\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[224:227], v[200:203], a[64:67], v112, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, 128\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[228:231], v[200:203], a[68:71], v113, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[232:235], v[200:203], a[72:75], v114, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s87, s87, 1\n\t" \
  "s_cmp_eq_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s85, 0x80000000, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[236:239], v[200:203], a[76:79], v115, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_and_b32 v122, s85, %[tail]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[236:239], v[204:207], a[108:111], v115, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_or3_b32 v120, s84, %[voa], v122\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[232:235], v[204:207], a[104:107], v114, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_or3_b32 v121, s84, %[vob], v122\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[228:231], v[204:207], a[100:103], v113, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[224:227], v[204:207], a[96:99], v112, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[240:243], v[204:207], a[112:115], v116, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v96, v127 offset:0\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[244:247], v[204:207], a[116:119], v117, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[248:251], v[204:207], a[120:123], v118, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v124, 0x10000, v124\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[252:255], v[204:207], a[124:127], v119, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[252:255], v[200:203], a[92:95], v119, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[248:251], v[200:203], a[88:91], v118, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v97, v127 offset:256\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[244:247], v[200:203], a[84:87], v117, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[240:243], v[200:203], a[80:83], v116, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[240:243], v[196:199], a[48:51], v116, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[244:247], v[196:199], a[52:55], v117, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v98, v127 offset:512\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[248:251], v[196:199], a[56:59], v118, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[252:255], v[196:199], a[60:63], v119, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[252:255], v[192:195], a[28:31], v119, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[248:251], v[192:195], a[24:27], v118, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[244:247], v[192:195], a[20:23], v117, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v99, v127 offset:768\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[240:243], v[192:195], a[16:19], v116, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[144:147], v[240:243], v[208:211], a[144:147], v116, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[148:151], v[244:247], v[208:211], a[148:151], v117, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[152:155], v[248:251], v[208:211], a[152:155], v118, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[156:159], v[252:255], v[208:211], a[156:159], v119, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[188:191], v[252:255], v[212:215], a[188:191], v119, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v100, v127 offset:1024\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[184:187], v[248:251], v[212:215], a[184:187], v118, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[180:183], v[244:247], v[212:215], a[180:183], v117, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[176:179], v[240:243], v[212:215], a[176:179], v116, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[208:211], v[240:243], v[216:219], a[208:211], v116, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v101, v127 offset:1280\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[212:215], v[244:247], v[216:219], a[212:215], v117, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[216:219], v[248:251], v[216:219], a[216:219], v118, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[220:223], v[252:255], v[216:219], a[220:223], v119, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[252:255], v[252:255], v[220:223], a[252:255], v119, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[248:251], v[248:251], v[220:223], a[248:251], v118, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v102, v127 offset:1536\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[244:247], v[244:247], v[220:223], a[244:247], v117, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[240:243], v[240:243], v[220:223], a[240:243], v116, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[236:239], v[236:239], v[220:223], a[236:239], v115, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[232:235], v[232:235], v[220:223], a[232:235], v114, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v103, v127 offset:1792\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[228:231], v[228:231], v[220:223], a[228:231], v113, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[224:227], v[224:227], v[220:223], a[224:227], v112, v111 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v125, 0x10000, v125\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[192:195], v[224:227], v[216:219], a[192:195], v112, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[196:199], v[228:231], v[216:219], a[196:199], v113, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[200:203], v[232:235], v[216:219], a[200:203], v114, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[204:207], v[236:239], v[216:219], a[204:207], v115, v110 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[172:175], v[236:239], v[212:215], a[172:175], v115, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[168:171], v[232:235], v[212:215], a[168:171], v114, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[164:167], v[228:231], v[212:215], a[164:167], v113, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[160:163], v[224:227], v[212:215], a[160:163], v112, v109 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[128:131], v[224:227], v[208:211], a[128:131], v112, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[132:135], v[228:231], v[208:211], a[132:135], v113, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[136:139], v[232:235], v[208:211], a[136:139], v114, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[140:143], v[236:239], v[208:211], a[140:143], v115, v108 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "L_sk_end%=:\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_LOOP_MX_LOW \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_add_u32 s81, %[ga0], 128\n\t" \
  "s_add_u32 s82, %[gb0], 128\n\t" \
  "s_mov_b32 s88, %[el]\n\t" \
  "s_mov_b32 s89, %[eka]\n\t" \
  "s_mov_b32 s90, %[ekb]\n\t" \
  "v_xor_b32 v124, 16, %[ra0]\n\t" \
  "v_xor_b32 v125, 16, %[rb0]\n\t" \
  "v_mov_b32 v126, %[rda]\n\t" \
  "v_mov_b32 v127, %[rdb]\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "s_add_u32 s87, s87, 1\n\t" \
  "s_cmp_eq_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s85, 0x80000000, 0\n\t" \
  "v_and_b32 v122, s85, %[tail]\n\t" \
  "v_or3_b32 v120, s84, %[voa], v122\n\t" \
  "v_or3_b32 v121, s84, %[vob], v122\n\t" \
  "s_waitcnt vmcnt(8)\n\t" \
  "s_barrier\n\t" \
  "ds_read_u16 v88, v126 offset:0\n\t" \
  "ds_read_u16 v89, v126 offset:256\n\t" \
  "ds_read_u16 v90, v126 offset:512\n\t" \
  "ds_read_u16 v91, v126 offset:768\n\t" \
  "ds_read_u16 v96, v127 offset:0\n\t" \
  "ds_read_u16 v97, v127 offset:256\n\t" \
  "ds_read_u16 v98, v127 offset:512\n\t" \
  "ds_read_u16 v99, v127 offset:768\n\t" \
  "ds_read_u16 v100, v127 offset:1024\n\t" \
  "ds_read_u16 v101, v127 offset:1280\n\t" \
  "ds_read_u16 v102, v127 offset:1536\n\t" \
  "ds_read_u16 v103, v127 offset:1792\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[160:163], v[128:131], a[0:3], v96, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[176:179], %[rb0] offset:8192\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[164:167], v[128:131], a[4:7], v97, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[180:183], %[rb0] offset:10240\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[168:171], v[128:131], a[8:11], v98, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[184:187], %[rb0] offset:12288\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[172:175], v[128:131], a[12:15], v99, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[188:191], %[rb0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[172:175], v[132:135], a[44:47], v99, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s82, %[gbs2]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[168:171], v[132:135], a[40:43], v98, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[192:195], v124 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[164:167], v[132:135], a[36:39], v97, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v104, v126 offset:8\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[160:163], v[132:135], a[32:35], v96, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[160:163], v[136:139], a[64:67], v96, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[224:227], v125 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[164:167], v[136:139], a[68:71], v97, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[168:171], v[136:139], a[72:75], v98, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[172:175], v[136:139], a[76:79], v99, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[228:231], v125 offset:2048\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[172:175], v[140:143], a[108:111], v99, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v105, v126 offset:264\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[168:171], v[140:143], a[104:107], v98, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[164:167], v[140:143], a[100:103], v97, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[232:235], v125 offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[160:163], v[140:143], a[96:99], v96, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[176:179], v[140:143], a[112:115], v100, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[180:183], v[140:143], a[116:119], v101, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[236:239], v125 offset:6144\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[184:187], v[140:143], a[120:123], v102, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v106, v126 offset:520\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[188:191], v[140:143], a[124:127], v103, v91 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 m0, s88\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[188:191], v[136:139], a[92:95], v103, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[196:199], v124 offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[184:187], v[136:139], a[88:91], v102, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[180:183], v[136:139], a[84:87], v101, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 %[vea], %[rea], s89 offen lds\n\t" \
  "s_add_u32 s89, s89, %[esa]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[176:179], v[136:139], a[80:83], v100, v90 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[200:203], v124 offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[176:179], v[132:135], a[48:51], v100, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v107, v126 offset:776\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[180:183], v[132:135], a[52:55], v101, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 m0, s88, 4096\n\t" \
  "s_xor_b32 s88, s88, 0x2000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[184:187], v[132:135], a[56:59], v102, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[204:207], v124 offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[188:191], v[132:135], a[60:63], v103, v89 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[188:191], v[128:131], a[28:31], v103, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 %[ve], %[reb], s90 offen lds\n\t" \
  "s_add_u32 s90, s90, %[esb]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[184:187], v[128:131], a[24:27], v102, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[180:183], v[128:131], a[20:23], v101, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[176:179], v[128:131], a[16:19], v100, v88 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt vmcnt(6) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[224:227], v[192:195], a[0:3], v96, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[240:243], v125 offset:8192\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, 128\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[228:231], v[192:195], a[4:7], v97, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[244:247], v125 offset:10240\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[232:235], v[192:195], a[8:11], v98, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[248:251], v125 offset:12288\n\t" \
  "s_add_u32 s87, s87, 1\n\t" \
  "s_cmp_eq_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s85, 0x80000000, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[236:239], v[192:195], a[12:15], v99, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[252:255], v125 offset:14336\n\t" \
  "v_and_b32 v122, s85, %[tail]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[236:239], v[196:199], a[44:47], v99, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_or3_b32 v120, s84, %[voa], v122\n\t" \
  "v_or3_b32 v121, s84, %[vob], v122\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[232:235], v[196:199], a[40:43], v98, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[228:231], v[196:199], a[36:39], v97, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[224:227], v[196:199], a[32:35], v96, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[224:227], v[200:203], a[64:67], v96, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v112, v127 offset:8\n\t" \
  "ds_read_u16 v113, v127 offset:264\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[228:231], v[200:203], a[68:71], v97, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[232:235], v[200:203], a[72:75], v98, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[236:239], v[200:203], a[76:79], v99, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v124, 0x10000, v124\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[236:239], v[204:207], a[108:111], v99, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[232:235], v[204:207], a[104:107], v98, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[228:231], v[204:207], a[100:103], v97, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v114, v127 offset:520\n\t" \
  "ds_read_u16 v115, v127 offset:776\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[224:227], v[204:207], a[96:99], v96, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[240:243], v[204:207], a[112:115], v100, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[244:247], v[204:207], a[116:119], v101, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[248:251], v[204:207], a[120:123], v102, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[252:255], v[204:207], a[124:127], v103, v91 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[252:255], v[200:203], a[92:95], v103, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v116, v127 offset:1032\n\t" \
  "ds_read_u16 v117, v127 offset:1288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[248:251], v[200:203], a[88:91], v102, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[244:247], v[200:203], a[84:87], v101, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[240:243], v[200:203], a[80:83], v100, v90 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v125, 0x10000, v125\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[240:243], v[196:199], a[48:51], v100, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[244:247], v[196:199], a[52:55], v101, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[248:251], v[196:199], a[56:59], v102, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v118, v127 offset:1544\n\t" \
  "ds_read_u16 v119, v127 offset:1800\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[252:255], v[196:199], a[60:63], v103, v89 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[252:255], v[192:195], a[28:31], v103, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[248:251], v[192:195], a[24:27], v102, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[244:247], v[192:195], a[20:23], v101, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[240:243], v[192:195], a[16:19], v100, v88 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc0 L_sk_end%=\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[160:163], v[128:131], a[0:3], v112, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[176:179], %[rb0] offset:8192\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[164:167], v[128:131], a[4:7], v113, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[180:183], %[rb0] offset:10240\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[168:171], v[128:131], a[8:11], v114, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[184:187], %[rb0] offset:12288\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[172:175], v[128:131], a[12:15], v115, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[188:191], %[rb0] offset:14336\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[172:175], v[132:135], a[44:47], v115, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v126, 0x2000, v126\n\t" \
  "v_xor_b32 v127, 0x2000, v127\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[168:171], v[132:135], a[40:43], v114, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s83, s82, %[gbs2]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[164:167], v[132:135], a[36:39], v113, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[192:195], v124 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[160:163], v[132:135], a[32:35], v112, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v88, v126 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[160:163], v[136:139], a[64:67], v112, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[224:227], v125 offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[164:167], v[136:139], a[68:71], v113, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[168:171], v[136:139], a[72:75], v114, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[172:175], v[136:139], a[76:79], v115, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[172:175], v[140:143], a[108:111], v115, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[228:231], v125 offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[168:171], v[140:143], a[104:107], v114, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v89, v126 offset:256\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[164:167], v[140:143], a[100:103], v113, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[232:235], v125 offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[160:163], v[140:143], a[96:99], v112, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[176:179], v[140:143], a[112:115], v116, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[180:183], v[140:143], a[116:119], v117, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[184:187], v[140:143], a[120:123], v118, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[236:239], v125 offset:6144\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[188:191], v[140:143], a[124:127], v119, v107 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v90, v126 offset:512\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[188:191], v[136:139], a[92:95], v119, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[184:187], v[136:139], a[88:91], v118, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[196:199], v124 offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[180:183], v[136:139], a[84:87], v117, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[176:179], v[136:139], a[80:83], v116, v106 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[176:179], v[132:135], a[48:51], v116, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[200:203], v124 offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[180:183], v[132:135], a[52:55], v117, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[184:187], v[132:135], a[56:59], v118, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v91, v126 offset:768\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[188:191], v[132:135], a[60:63], v119, v105 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[204:207], v124 offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[188:191], v[128:131], a[28:31], v119, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[184:187], v[128:131], a[24:27], v118, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[180:183], v[128:131], a[20:23], v117, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[176:179], v[128:131], a[16:19], v116, v104 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt vmcnt(4) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[224:227], v[192:195], a[0:3], v112, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[240:243], v125 offset:8192\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, 128\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[228:231], v[192:195], a[4:7], v113, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[244:247], v125 offset:10240\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[8:11], v[232:235], v[192:195], a[8:11], v114, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[248:251], v125 offset:12288\n\t" \
  "s_add_u32 s87, s87, 1\n\t" \
  "s_cmp_eq_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s85, 0x80000000, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[12:15], v[236:239], v[192:195], a[12:15], v115, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[252:255], v125 offset:14336\n\t" \
  "v_and_b32 v122, s85, %[tail]\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[44:47], v[236:239], v[196:199], a[44:47], v115, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_or3_b32 v120, s84, %[voa], v122\n\t" \
  "v_or3_b32 v121, s84, %[vob], v122\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[40:43], v[232:235], v[196:199], a[40:43], v114, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[36:39], v[228:231], v[196:199], a[36:39], v113, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[32:35], v[224:227], v[196:199], a[32:35], v112, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[64:67], v[224:227], v[200:203], a[64:67], v112, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v96, v127 offset:0\n\t" \
  "ds_read_u16 v97, v127 offset:256\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[68:71], v[228:231], v[200:203], a[68:71], v113, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[72:75], v[232:235], v[200:203], a[72:75], v114, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[76:79], v[236:239], v[200:203], a[76:79], v115, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v124, 0x10000, v124\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[108:111], v[236:239], v[204:207], a[108:111], v115, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[104:107], v[232:235], v[204:207], a[104:107], v114, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[100:103], v[228:231], v[204:207], a[100:103], v113, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v98, v127 offset:512\n\t" \
  "ds_read_u16 v99, v127 offset:768\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[96:99], v[224:227], v[204:207], a[96:99], v112, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[112:115], v[240:243], v[204:207], a[112:115], v116, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[116:119], v[244:247], v[204:207], a[116:119], v117, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[120:123], v[248:251], v[204:207], a[120:123], v118, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[124:127], v[252:255], v[204:207], a[124:127], v119, v107 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[92:95], v[252:255], v[200:203], a[92:95], v119, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v100, v127 offset:1024\n\t" \
  "ds_read_u16 v101, v127 offset:1280\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[88:91], v[248:251], v[200:203], a[88:91], v118, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[84:87], v[244:247], v[200:203], a[84:87], v117, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[80:83], v[240:243], v[200:203], a[80:83], v116, v106 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_xor_b32 v125, 0x10000, v125\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[48:51], v[240:243], v[196:199], a[48:51], v116, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[52:55], v[244:247], v[196:199], a[52:55], v117, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[56:59], v[248:251], v[196:199], a[56:59], v118, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_u16 v102, v127 offset:1536\n\t" \
  "ds_read_u16 v103, v127 offset:1792\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[60:63], v[252:255], v[196:199], a[60:63], v119, v105 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[28:31], v[252:255], v[192:195], a[28:31], v119, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[24:27], v[248:251], v[192:195], a[24:27], v118, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[20:23], v[244:247], v[192:195], a[20:23], v117, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "v_mfma_scale_f32_16x16x128_f8f6f4 a[16:19], v[240:243], v[192:195], a[16:19], v116, v104 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "L_sk_end%=:\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_CLOBBERS_MX \
  "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15", \
  "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31", \
  "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", \
  "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", \
  "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79", \
  "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95", \
  "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", \
  "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127", \
  "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", "a140", "a141", "a142", "a143", \
  "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", "a159", \
  "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", "a172", "a173", "a174", "a175", \
  "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191", \
  "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", "a204", "a205", "a206", "a207", \
  "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223", \
  "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", "a236", "a237", "a238", "a239", \
  "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255", \
  "v88", "v89", "v90", "v91", "v92", "v93", "v94", "v95", "v96", "v97", "v98", "v99", "v100", "v101", "v102", "v103", \
  "v104", "v105", "v106", "v107", "v108", "v109", "v110", "v111", "v112", "v113", "v114", "v115", "v116", "v117", "v118", "v119", \
  "v120", "v121", "v122", "v123", "v124", "v125", "v126", "v127", "v128", "v129", "v130", "v131", "v132", "v133", "v134", "v135", \
  "v136", "v137", "v138", "v139", "v140", "v141", "v142", "v143", "v144", "v145", "v146", "v147", "v148", "v149", "v150", "v151", \
  "v152", "v153", "v154", "v155", "v156", "v157", "v158", "v159", "v160", "v161", "v162", "v163", "v164", "v165", "v166", "v167", \
  "v168", "v169", "v170", "v171", "v172", "v173", "v174", "v175", "v176", "v177", "v178", "v179", "v180", "v181", "v182", "v183", \
  "v184", "v185", "v186", "v187", "v188", "v189", "v190", "v191", "v192", "v193", "v194", "v195", "v196", "v197", "v198", "v199", \
  "v200", "v201", "v202", "v203", "v204", "v205", "v206", "v207", "v208", "v209", "v210", "v211", "v212", "v213", "v214", "v215", \
  "v216", "v217", "v218", "v219", "v220", "v221", "v222", "v223", "v224", "v225", "v226", "v227", "v228", "v229", "v230", "v231", \
  "v232", "v233", "v234", "v235", "v236", "v237", "v238", "v239", "v240", "v241", "v242", "v243", "v244", "v245", "v246", "v247", \
  "v248", "v249", "v250", "v251", "v252", "v253", "v254", "v255", "s80", "s81", "s82", "s83", "s84", "s85", "s86", "s87", \
  "s88", "s89", "s90"
