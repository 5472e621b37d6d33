// The gfx950 code objects built from kernels.hip, ingest.hip, prompt.hip,
// serve.hip and rows.hip, linked into the library as read-only data and loaded with hipModuleLoadData at init.
    .section .rodata
    .balign 4096
    .global sml_code_object
    .type sml_code_object, @object
sml_code_object:
    .incbin "kernels.hsaco"
    .global sml_code_object_end
sml_code_object_end:
    .byte 0
    .balign 4096
    .global sml_ingest_object
    .type sml_ingest_object, @object
sml_ingest_object:
    .incbin "ingest.hsaco"
    .global sml_ingest_object_end
sml_ingest_object_end:
    .byte 0
    .balign 4096
    .global sml_prompt_object
    .type sml_prompt_object, @object
sml_prompt_object:
    .incbin "prompt.hsaco"
    .global sml_prompt_object_end
sml_prompt_object_end:
    .byte 0
    .balign 4096
    .global sml_serve_object
    .type sml_serve_object, @object
sml_serve_object:
    .incbin "serve.hsaco"
    .global sml_serve_object_end
sml_serve_object_end:
    .byte 0
    .balign 4096
    .global sml_rows_object
    .type sml_rows_object, @object
sml_rows_object:
    .incbin "rows.hsaco"
    .global sml_rows_object_end
sml_rows_object_end:
    .byte 0
    .section .note.GNU-stack,"",@progbits
